// Root-mean-square norm of the rows of a matrix, with the residual's addition in front and an 8-bit output behind, and its
// gradient.
//   h = src + residual            (written in src's type where that is wanted; what follows takes the unrounded sum)
//   y = h r w,  r = 1 / sqrt(mean h^2 + eps)
//   8 bits: q = round(y / s), saturated; s is given (one for all), or made: largest |y| of the row, or of each group of
//   its columns, over 127 (s8) or 448 (e4m3).  A largest value below 1e-36 makes s = 0 and q = 0; a NaN makes s NaN.
// Gradient, with z = w dy:
//   dh = r z - h r^3 mean(h z) (+ the gradient that comes along the residual path),  dw = sum over the rows of dy h r
//
// Bound by memory.  A row stays in the registers of a CTA (of a warp where it is short), so each tensor crosses memory once;
// sums are f32: in a thread, over the warp, over the CTA.  A thread holds chunks of eight columns: neighbours in 16-byte
// accesses, or 32 apart where rows start anywhere.
#include <cuda_fp8.h>

#include <algorithm>

#include "launch.h"
#include "token_rows.cuh"

namespace qmm {

namespace {

constexpr float SMALLEST_MAX = 1e-36f; // 448 / this is still finite

__device__ __forceinline__ uint32_t cvt_s8(float v) { // saturated, to nearest even; 0 for a NaN
    int r;
    asm("cvt.rni.sat.s8.f32 %0, %1;" : "=r"(r) : "f"(v));
    return (uint32_t)r & 0xffu;
}
__device__ __forceinline__ uint32_t cvt_e4m3x2(float lo, float hi) { // saturated at 448
    return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}

// Eight columns of a row.  VEC: neighbours from `col` on, the row a multiple of eight and all its tensors aligned to 16 bytes
// (8-bit ones to 8).  Otherwise col, col + 32, ...: a warp covers the same 256 columns in either form.
template <bool VEC> __device__ __forceinline__ int64_t chunk_column(int64_t chunk) {
    return VEC ? chunk * 8 : chunk / 32 * 256 + chunk % 32;
}
template <typename T, bool VEC> struct Chunk {
    uint4 raw[VEC ? sizeof(T) / 2 : 1];
    T each[VEC ? 1 : 8];
    __device__ __forceinline__ void load(const T *row, int64_t col, int64_t cols) {
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
                raw[i] = make_uint4(0, 0, 0, 0);
                if (col < cols) raw[i] = ptx::ld_dependent((const uint4 *)(row + col) + i);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) each[i] = col + 32 * i < cols ? row[col + 32 * i] : from_f32<T>(0.f);
        }
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        if constexpr (!VEC) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = to_f32(each[i]);
        } else if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                v[4 * i] = __uint_as_float(raw[i].x);
                v[4 * i + 1] = __uint_as_float(raw[i].y);
                v[4 * i + 2] = __uint_as_float(raw[i].z);
                v[4 * i + 3] = __uint_as_float(raw[i].w);
            }
        } else {
            unpack2(raw[0].x, v[0], v[1], T());
            unpack2(raw[0].y, v[2], v[3], T());
            unpack2(raw[0].z, v[4], v[5], T());
            unpack2(raw[0].w, v[6], v[7], T());
        }
    }
    static __device__ __forceinline__ void store(T *row, int64_t col, int64_t cols, const float (&v)[8]) {
        if constexpr (VEC) {
            Cols<T, true>::store(row, col, cols, v);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (col + 32 * i < cols) row[col + 32 * i] = from_f32<T>(v[i]);
        }
    }
};

template <typename T, bool VEC>
__device__ __forceinline__ void load_weights(const NormArgs &a, int64_t col, float (&w)[8]) {
    if (!a.weights) {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = 1.f;
    } else if (a.weights_dt == DT_F32) {
        Chunk<float, VEC> c;
        c.load((const float *)a.weights, col, a.cols);
        c.get(w);
    } else {
        Chunk<T, VEC> c;
        c.load((const T *)a.weights, col, a.cols);
        c.get(w);
    }
}

template <bool VEC> __device__ __forceinline__ void store_8bit(const NormArgs &a, int64_t t, int64_t col, const float (&v)[8]) {
    uint8_t *row = (uint8_t *)a.dst + t * a.dst_ld;
    if (col >= a.cols) return;
    uint32_t lo, hi; // bytes 0 to 3 and 4 to 7
    if (a.dst_dt == DT_S8) {
        lo = cvt_s8(v[0]) | cvt_s8(v[1]) << 8 | cvt_s8(v[2]) << 16 | cvt_s8(v[3]) << 24;
        hi = cvt_s8(v[4]) | cvt_s8(v[5]) << 8 | cvt_s8(v[6]) << 16 | cvt_s8(v[7]) << 24;
    } else {
        lo = cvt_e4m3x2(v[0], v[1]) | cvt_e4m3x2(v[2], v[3]) << 16;
        hi = cvt_e4m3x2(v[4], v[5]) | cvt_e4m3x2(v[6], v[7]) << 16;
    }
    if constexpr (VEC) {
        *reinterpret_cast<uint2 *>(row + col) = make_uint2(lo, hi);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (col + 32 * i < a.cols) row[col + 32 * i] = (uint8_t)((i < 4 ? lo : hi) >> 8 * (i % 4));
    }
}

// Sum (of one or two numbers), or largest of unsigned bits, over the threads that share a row.  `buffer`: 64 words of shared
// memory that nothing else uses until the next barrier but one.
template <int THREADS, int N> __device__ __forceinline__ void row_sum(float (&v)[N], float *buffer) {
#pragma unroll
    for (int s = 16; s > 0; s /= 2)
#pragma unroll
        for (int n = 0; n < N; ++n) v[n] += __shfl_xor_sync(0xffffffffu, v[n], s);
    if constexpr (THREADS > 32) {
        const int lane = threadIdx.x & 31;
        if (lane == 0)
#pragma unroll
            for (int n = 0; n < N; ++n) buffer[n * 32 + threadIdx.x / 32] = v[n];
        __syncthreads();
#pragma unroll
        for (int n = 0; n < N; ++n) {
            v[n] = lane < THREADS / 32 ? buffer[n * 32 + lane] : 0.f;
#pragma unroll
            for (int s = THREADS / 64; s > 0; s /= 2) v[n] += __shfl_xor_sync(0xffffffffu, v[n], s);
            v[n] = __shfl_sync(0xffffffffu, v[n], 0);
        }
    }
}
template <int THREADS> __device__ __forceinline__ uint32_t row_max(uint32_t v, uint32_t *buffer) {
    v = __reduce_max_sync(0xffffffffu, v);
    if constexpr (THREADS > 32) {
        const int lane = threadIdx.x & 31;
        if (lane == 0) buffer[threadIdx.x / 32] = v;
        __syncthreads();
        v = __reduce_max_sync(0xffffffffu, lane < THREADS / 32 ? buffer[lane] : 0u);
    }
    return v;
}

// scale and its reciprocal from the bits of the largest |value| (the bits of a NaN are above all others)
__device__ __forceinline__ float make_scale(uint32_t most, float limit, float &inverse) {
    const float m = __uint_as_float(most);
    inverse = m < SMALLEST_MAX ? 0.f : limit / m;
    return m < SMALLEST_MAX ? 0.f : m / limit;
}

// v / scale of its group, and the scales.  Groups of 16 to 256 columns, a power of two: in a warp's 256 columns they are whole
// lanes' (VEC), or one to eight times 32 columns of all lanes, or half of them.
template <bool VEC> __device__ __forceinline__ void scale_groups(const NormArgs &a, int64_t t, int64_t col, float limit, float (&v)[8]) {
    float *scales = a.scales + t * (a.cols / a.group);
    float inverse;
    if constexpr (VEC) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
        for (int s = 1; s < a.group / 8; s *= 2) m = max(m, __shfl_xor_sync(0xffffffffu, m, s));
        const float s = make_scale(m, limit, inverse);
        if (col < a.cols && (col & (a.group - 1)) == 0) scales[col / a.group] = s;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= inverse;
    } else {
        uint32_t m[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            m[i] = __float_as_uint(v[i]) & 0x7fffffffu;
            if (a.group == 16) {
#pragma unroll
                for (int s = 1; s < 16; s *= 2) m[i] = max(m[i], __shfl_xor_sync(0xffffffffu, m[i], s));
            } else {
                m[i] = __reduce_max_sync(0xffffffffu, m[i]);
            }
        }
#pragma unroll
        for (int step = 1; step < 8; step *= 2) // (pairs, fours, all eight of the 32 columns)
            if (a.group > 32 * step) {
                uint32_t other[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) other[i] = m[i ^ step];
#pragma unroll
                for (int i = 0; i < 8; ++i) m[i] = max(m[i], other[i]);
            }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float s = make_scale(m[i], limit, inverse);
            if (col + 32 * i < a.cols && ((col + 32 * i) & (a.group - 1)) == 0) scales[(col + 32 * i) / a.group] = s;
            v[i] *= inverse;
        }
    }
}

// A CTA's threads, the rows that they work on at the same time, and the CTAs of an SM that registers are cut to.
template <int THREADS> constexpr int BLOCK = THREADS == 32 ? 256 : THREADS;
template <int THREADS> constexpr int TEAMS = THREADS == 32 ? 8 : 1;
template <typename T, bool VEC, int THREADS> constexpr int FORWARD_CTAS = THREADS > 256 ? 1 : (VEC && sizeof(T) == 2 ? 768 : 512) / BLOCK<THREADS>;
template <int THREADS> constexpr int BACKWARD_CTAS = THREADS > 256 ? 1 : 512 / BLOCK<THREADS>;
template <int CHUNKS> constexpr bool AHEAD = CHUNKS <= 2; // registers for a row that is on its way

// CTAs that stay take rows in turn; the next row is on its way while one is worked on, and the weights stay in registers.
template <typename T, bool VEC, int THREADS, int CHUNKS>
__global__ void __launch_bounds__(BLOCK<THREADS>, FORWARD_CTAS<T, VEC, THREADS>) rms_norm_kernel(const __grid_constant__ NormArgs a) {
    __shared__ float sums[2][64];
    __shared__ uint32_t largest[2][32];
    ptx::grid_dependency_wait();
    const int thread = threadIdx.x % THREADS;
    const int64_t step = (int64_t)gridDim.x * TEAMS<THREADS>;
    int64_t t = (int64_t)blockIdx.x * TEAMS<THREADS> + (THREADS == 32 ? threadIdx.x / 32 : 0);
    Chunk<T, VEC> x[CHUNKS], r[CHUNKS];
    auto load = [&](int64_t row) {
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const int64_t col = chunk_column<VEC>(c * THREADS + thread);
            x[c].load((const T *)a.src + row * a.src_ld, col, a.cols);
            if (a.residual) r[c].load((const T *)a.residual + row * a.residual_ld, col, a.cols);
        }
    };
    if (AHEAD<CHUNKS> && t < a.rows) load(t);
    float w[CHUNKS][8];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) load_weights<T, VEC>(a, chunk_column<VEC>(c * THREADS + thread), w[c]);
    const float given = a.scaling == NORM_SCALE_GIVEN ? ptx::ld_dependent(a.scales) : 1.f;
    const float limit = a.dst_dt == DT_S8 ? 127.f : 448.f;
    for (int turn = 0; t < a.rows; t += step, turn ^= 1) {
        if (!AHEAD<CHUNKS>) load(t);
        float h[CHUNKS][8];
        float sum[1] = {0.f};
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            x[c].get(h[c]);
            if (a.residual) {
                float v[8];
                r[c].get(v);
#pragma unroll
                for (int i = 0; i < 8; ++i) h[c][i] += v[i];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[0] = fmaf(h[c][i], h[c][i], sum[0]);
        }
        if (AHEAD<CHUNKS> && t + step < a.rows) load(t + step);
        if (a.sum) {
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c) Chunk<T, VEC>::store((T *)a.sum + t * a.sum_ld, chunk_column<VEC>(c * THREADS + thread), a.cols, h[c]);
        }
        row_sum<THREADS>(sum, sums[turn]);
        const float scale = 1.f / sqrtf(sum[0] / (float)a.cols + a.epsilon);
        uint32_t most = 0;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                h[c][i] = h[c][i] * scale * w[c][i];
                most = max(most, __float_as_uint(h[c][i]) & 0x7fffffffu);
            }
        float inverse = 1.f / given;
        if (a.scaling == NORM_SCALE_ROW) {
            const float s = make_scale(row_max<THREADS>(most, largest[turn]), limit, inverse);
            if (thread == 0) a.scales[t] = s;
        }
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const int64_t col = chunk_column<VEC>(c * THREADS + thread);
            if (a.scaling == NORM_SCALE_GROUP) {
                scale_groups<VEC>(a, t, col, limit, h[c]);
            } else if (a.scaling != NORM_SCALE_NONE) {
#pragma unroll
                for (int i = 0; i < 8; ++i) h[c][i] *= inverse;
            }
            switch (a.dst_dt) {
                case DT_F32: Chunk<float, VEC>::store((float *)a.dst + t * a.dst_ld, col, a.cols, h[c]); break;
                case DT_BF16: Chunk<__nv_bfloat16, VEC>::store((__nv_bfloat16 *)a.dst + t * a.dst_ld, col, a.cols, h[c]); break;
                case DT_F16: Chunk<__half, VEC>::store((__half *)a.dst + t * a.dst_ld, col, a.cols, h[c]); break;
                default: store_8bit<VEC>(a, t, col, h[c]);
            }
        }
    }
}

// Gradient: CTAs that stay take rows in turn; the weights and this CTA's part of their gradient stay in registers, and the
// parts of all CTAs meet in the scratchpad, which the kernel behind this one adds up, in the same order every time.
template <typename T, bool VEC, int THREADS, int CHUNKS>
__global__ void __launch_bounds__(BLOCK<THREADS>, BACKWARD_CTAS<THREADS>) rms_norm_backward_kernel(const __grid_constant__ NormArgs a) {
    extern __shared__ float gathered[]; // a warp a row: [8][columns]
    __shared__ float sums[2][64];
    ptx::grid_dependency_wait();
    const int thread = threadIdx.x % THREADS, team = THREADS == 32 ? threadIdx.x / 32 : 0;
    const int64_t step = (int64_t)gridDim.x * TEAMS<THREADS>;
    int64_t t = (int64_t)blockIdx.x * TEAMS<THREADS> + team;
    Chunk<T, VEC> next_h[CHUNKS], next_dy[CHUNKS], next_more[CHUNKS];
    auto load = [&](int64_t row) {
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const int64_t col = chunk_column<VEC>(c * THREADS + thread);
            next_h[c].load((const T *)a.src + row * a.src_ld, col, a.cols);
            next_dy[c].load((const T *)a.diff_dst + row * a.diff_dst_ld, col, a.cols);
            if (a.residual) next_more[c].load((const T *)a.residual + row * a.residual_ld, col, a.cols);
        }
    };
    if (AHEAD<CHUNKS> && t < a.rows) load(t);
    float w[CHUNKS][8], dw[CHUNKS][8];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
        load_weights<T, VEC>(a, chunk_column<VEC>(c * THREADS + thread), w[c]);
#pragma unroll
        for (int i = 0; i < 8; ++i) dw[c][i] = 0.f;
    }
    for (int turn = 0; t < a.rows; t += step, turn ^= 1) {
        if (!AHEAD<CHUNKS>) load(t);
        Chunk<T, VEC> h[CHUNKS], dy[CHUNKS], more[CHUNKS];
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            h[c] = next_h[c];
            dy[c] = next_dy[c];
            if (a.residual) more[c] = next_more[c];
        }
        if (AHEAD<CHUNKS> && t + step < a.rows) load(t + step);
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            float x[8], g[8];
            h[c].get(x);
            dy[c].get(g);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                s[0] = fmaf(x[i], x[i], s[0]);
                s[1] = fmaf(x[i] * w[c][i], g[i], s[1]);
            }
        }
        row_sum<THREADS>(s, sums[turn]);
        const float r = 1.f / sqrtf(s[0] / (float)a.cols + a.epsilon);
        const float inner = s[1] / (float)a.cols * r * r; // dh = r (z - h inner)
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            float x[8], g[8], d[8];
            h[c].get(x);
            dy[c].get(g);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                d[i] = r * fmaf(g[i], w[c][i], -x[i] * inner);
                dw[c][i] = fmaf(g[i], x[i] * r, dw[c][i]);
            }
            if (a.residual) {
                more[c].get(x);
#pragma unroll
                for (int i = 0; i < 8; ++i) d[i] += x[i];
            }
            Chunk<T, VEC>::store((T *)a.diff_src + t * a.diff_src_ld, chunk_column<VEC>(c * THREADS + thread), a.cols, d);
        }
    }
    asm volatile("griddepcontrol.launch_dependents;"); // nothing is read any more
    if (!a.parts) return;
    if constexpr (THREADS == 32) {
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) Chunk<float, VEC>::store(gathered + team * a.cols, chunk_column<VEC>(c * 32 + thread), a.cols, dw[c]);
        __syncthreads();
        for (int col = threadIdx.x; col < (int)a.cols; col += 256) {
            float sum = 0.f;
#pragma unroll
            for (int q = 0; q < 8; ++q) sum += gathered[q * a.cols + col];
            a.parts[blockIdx.x * a.cols + col] = sum;
        }
    } else {
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c)
            Chunk<float, VEC>::store(a.parts + blockIdx.x * a.cols, chunk_column<VEC>(c * THREADS + thread), a.cols, dw[c]);
    }
}

// diff_weights[col] = sum of the parts: 32 columns a CTA, its warps take the parts in turn
__global__ void __launch_bounds__(1024) rms_norm_weights_kernel(const __grid_constant__ NormArgs a) {
    __shared__ float sums[32][33];
    ptx::grid_dependency_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    const int64_t col = (int64_t)blockIdx.x * 32 + lane;
    float sum = 0.f;
    if (col < a.cols)
        for (int p = warp; p < a.part_count; p += 32) sum += ptx::ld_dependent(a.parts + p * a.cols + col);
    sums[warp][lane] = sum;
    __syncthreads();
    sum = sums[lane][warp];
#pragma unroll
    for (int s = 16; s > 0; s /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, s);
    const int64_t mine = (int64_t)blockIdx.x * 32 + warp;
    if (lane == 0 && mine < a.cols) {
        if (a.weights_grad_dt == DT_F32) ((float *)a.diff_weights)[mine] = sum;
        else if (a.weights_grad_dt == DT_BF16) ((__nv_bfloat16 *)a.diff_weights)[mine] = __float2bfloat16_rn(sum);
        else ((__half *)a.diff_weights)[mine] = __float2half_rn(sum);
    }
}

template <typename T, bool VEC, int THREADS, int CHUNKS> int launch_shape(NormArgs &a, bool backward, int sm_count, cudaStream_t st) {
    const int64_t ctas = (a.rows + TEAMS<THREADS> - 1) / TEAMS<THREADS>;
    if (!backward)
        return launch_dependent(rms_norm_kernel<T, VEC, THREADS, CHUNKS>, a, (unsigned)std::min<int64_t>(ctas, sm_count * FORWARD_CTAS<T, VEC, THREADS>),
                BLOCK<THREADS>, 0, st);
    // a part of the weights' gradient for each CTA: four rows at least, unless the SMs are too many
    a.part_count = (int)std::min<int64_t>(std::min<int64_t>(ctas, std::max<int64_t>(ctas / 4, sm_count)), sm_count * norm_gradient_ctas(a.cols));
    return launch_dependent(rms_norm_backward_kernel<T, VEC, THREADS, CHUNKS>, a, a.part_count, BLOCK<THREADS>,
            THREADS == 32 ? 8 * a.cols * sizeof(float) : 0, st);
}
// Threads of a row and its chunks of eight columns each: two chunks keep enough loads in flight, more where a CTA has no more threads.
template <typename T, bool VEC> int launch_form(NormArgs &a, bool backward, int sm_count, cudaStream_t st) {
    const int64_t chunks = VEC ? (a.cols + 7) / 8 : (a.cols + 255) / 256 * 32;
    if (chunks <= 32) return launch_shape<T, VEC, 32, 1>(a, backward, sm_count, st);
    if (chunks <= 64) return launch_shape<T, VEC, 32, 2>(a, backward, sm_count, st);
    if (chunks <= 128) return launch_shape<T, VEC, 64, 2>(a, backward, sm_count, st);
    if (chunks <= 256) return launch_shape<T, VEC, 128, 2>(a, backward, sm_count, st);
    if (chunks <= 512) return launch_shape<T, VEC, 256, 2>(a, backward, sm_count, st);
    if (chunks <= 1024) return launch_shape<T, VEC, 512, 2>(a, backward, sm_count, st);
    return launch_shape<T, VEC, 512, 4>(a, backward, sm_count, st);
}

template <typename T> int launch_typed(NormArgs a, bool backward, int sm_count, cudaStream_t st) {
    const int64_t size = sizeof(T);
    bool vec = a.cols % 8 == 0 && rows_aligned(a.src, a.src_ld * size, a.rows)
            && (!a.residual || rows_aligned(a.residual, a.residual_ld * size, a.rows)) && (uintptr_t)a.weights % 16 == 0;
    if (backward) {
        vec = vec && rows_aligned(a.diff_dst, a.diff_dst_ld * size, a.rows) && rows_aligned(a.diff_src, a.diff_src_ld * size, a.rows);
    } else {
        const int64_t out = a.dst_dt == DT_F32 ? 4 : a.dst_dt == DT_BF16 || a.dst_dt == DT_F16 ? 2 : 1;
        vec = vec && (!a.sum || rows_aligned(a.sum, a.sum_ld * size, a.rows))
                && (out > 1 ? rows_aligned(a.dst, a.dst_ld * out, a.rows) : (uintptr_t)a.dst % 8 == 0 && (a.rows <= 1 || a.dst_ld % 8 == 0));
    }
    int rc = vec ? launch_form<T, true>(a, backward, sm_count, st) : launch_form<T, false>(a, backward, sm_count, st);
    if (rc == 0) count_launch();
    if (rc == 0 && a.diff_weights) {
        rc = launch_dependent(rms_norm_weights_kernel, a, (unsigned)((a.cols + 31) / 32), 1024, 0, st);
        if (rc == 0) count_launch();
    }
    return rc;
}

int launch_any(const NormArgs &a, bool backward, int sm_count, cudaStream_t st) {
    switch (a.dt) {
        case DT_F32: return launch_typed<float>(a, backward, sm_count, st);
        case DT_BF16: return launch_typed<__nv_bfloat16>(a, backward, sm_count, st);
        case DT_F16: return launch_typed<__half>(a, backward, sm_count, st);
        default: return 3;
    }
}

} // namespace

// CTAs per SM of the gradient's kernel, each with a part of the weights' gradient
int norm_gradient_ctas(int64_t cols) { return cols <= 512 ? 2 : cols <= 1024 ? 8 : cols <= 2048 ? 4 : cols <= 4096 ? 2 : 1; }
size_t norm_scratch_bytes(int64_t cols, int sm_count) { return (size_t)sm_count * norm_gradient_ctas(cols) * cols * sizeof(float); }

int launch_rms_norm(const NormArgs &a, int sm_count, cudaStream_t st) {
    if (a.rows == 0 || a.cols == 0) return 0;
    return launch_any(a, false, sm_count, st);
}
int launch_rms_norm_backward(const NormArgs &a, int sm_count, cudaStream_t st) {
    if (a.cols == 0) return 0;
    if (a.rows == 0) { // no rows: a weights' gradient of zeros
        if (!a.diff_weights) return 0;
        NormArgs none = a;
        none.part_count = 0;
        const int rc = launch_dependent(rms_norm_weights_kernel, none, (unsigned)((a.cols + 31) / 32), 1024, 0, st);
        if (rc == 0) count_launch();
        return rc;
    }
    return launch_any(a, true, sm_count, st);
}

} // namespace qmm

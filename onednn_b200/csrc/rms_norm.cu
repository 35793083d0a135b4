// Root-mean-square norm of the rows of a matrix, with the residual's addition in front and an 8-bit output behind, and its
// gradient.
//   h = src + residual            (written in src's type where that is wanted; what follows takes the unrounded sum)
//   y = h r w,  r = 1 / sqrt(mean h^2 + eps)
//   8 bits: q = round(y / s), saturated; s is given (one for all), or made: largest |y| of the row, or of each group of
//   its columns, over 127 (s8) or 448 (e4m3).  A largest value below 1.4e-36 makes s = 0 and q = 0; a NaN makes s NaN.
// Gradient, with z = w dy:
//   dh = r z - h r^3 mean(h z) (+ the gradient that comes along the residual path),  dw = sum over the rows of dy h r
//
// Bound by memory where rows are many and aligned.  A row stays in the registers of a CTA (of a warp where it is short), so each
// tensor crosses memory once; sums are f32: in a thread (two columns an instruction), over the warp, over the CTA.  A thread holds
// chunks of eight columns: neighbours in 16-byte accesses, or 32 apart where rows start anywhere.
// us a call (floor): 8192 x 4096 bf16 with residual and sum to e4m3 37.7 (35.8, 6.2 TB/s); 4099 x 4096 bf16 to e4m3 with scales of
// 128 columns 17.2 (7.8; some 630 instructions a warp and row, at odd starts 25.6), with one scale 13.2; 2048 x 5120 bf16 with residual and
// sum, a scale a row 15.5 (11.2); 3001 x 2047 f16 at odd starts 14.6 (7.5; accesses of two bytes).  Gradient: 8192 x 4096 bf16 with the
// residual's 48 (40.9), 8192 x 1024 17.2 (10.2), 1021 x 1367 f32 at odd starts 8.3 (2.6), of which 2 to 3 are the second kernel.
#include <cuda_fp8.h>

#include <algorithm>

#include "launch.h"
#include "token_rows.cuh"

namespace qmm {

namespace {

constexpr float SMALLEST_MAX = 1.4e-36f; // 448 / this is still finite

__device__ __forceinline__ uint32_t cvt_s8(float v) { // saturated, to nearest even; 0 for a NaN
    int r;
    asm("cvt.rni.sat.s8.f32 %0, %1;" : "=r"(r) : "f"(v));
    return (uint32_t)r & 0xffu;
}
__device__ __forceinline__ uint32_t cvt_e4m3x2(float lo, float hi) { // saturated at 448
    return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}

// two 32-bit floats in a register pair: one instruction works on both
struct Pair { uint64_t bits; };
__device__ __forceinline__ Pair pair(float lo, float hi) {
    Pair r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.bits) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ Pair both(float v) { return pair(v, v); }
__device__ __forceinline__ void split(Pair p, float &lo, float &hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(p.bits)); }
__device__ __forceinline__ Pair operator*(Pair a, Pair b) {
    Pair r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits));
    return r;
}
__device__ __forceinline__ Pair operator+(Pair a, Pair b) {
    Pair r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits));
    return r;
}
__device__ __forceinline__ Pair fma(Pair a, Pair b, Pair c) {
    Pair r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits), "l"(c.bits));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) { // NaN if either is
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// Eight columns of a row.  VEC: neighbours from `col` on, the row a multiple of eight and all its tensors aligned to 16 bytes
// (8-bit ones to 8).  Otherwise col, col + 32, ...: a warp covers the same 256 columns in either form.
template <bool VEC> __device__ __forceinline__ int chunk_column(int chunk) {
    return VEC ? chunk * 8 : chunk / 32 * 256 + chunk % 32;
}
template <typename T, bool VEC> struct Chunk {
    uint4 raw[VEC ? sizeof(T) / 2 : 1];
    T each[VEC ? 1 : 8];
    __device__ __forceinline__ void load(const T *row, int col, int cols) {
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
                raw[i] = make_uint4(0, 0, 0, 0);
                if (col < cols) raw[i] = ptx::ld_dependent((const uint4 *)(row + col) + i);
            }
        } else if (col + 224 < cols) {
#pragma unroll
            for (int i = 0; i < 8; ++i) each[i] = row[col + 32 * i];
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
    __device__ __forceinline__ void get(Pair (&p)[4]) const {
        float v[8];
        get(v);
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = pair(v[2 * i], v[2 * i + 1]);
    }
    static __device__ __forceinline__ void store(T *row, int col, int cols, const Pair (&p)[4]) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) split(p[i], v[2 * i], v[2 * i + 1]);
        if constexpr (VEC) {
            Cols<T, true>::store(row, col, cols, v);
        } else if (col + 224 < cols) {
#pragma unroll
            for (int i = 0; i < 8; ++i) row[col + 32 * i] = from_f32<T>(v[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (col + 32 * i < cols) row[col + 32 * i] = from_f32<T>(v[i]);
        }
    }
};

template <typename T, bool VEC>
__device__ __forceinline__ void load_weights(const NormArgs &a, int col, Pair (&w)[4]) {
    if (!a.weights) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = both(1.f);
    } else if (a.weights_dt == DT_F32) {
        Chunk<float, VEC> c;
        c.load((const float *)a.weights, col, (int)a.cols);
        c.get(w);
    } else {
        Chunk<T, VEC> c;
        c.load((const T *)a.weights, col, (int)a.cols);
        c.get(w);
    }
}

template <bool VEC> __device__ __forceinline__ void store_8bit(const NormArgs &a, uint32_t t, int col, const Pair (&p)[4]) {
    uint8_t *row = (uint8_t *)a.dst + t * a.dst_ld;
    const int cols = (int)a.cols;
    if (col >= cols) return;
    float v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) split(p[i], v[2 * i], v[2 * i + 1]);
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
            if (col + 32 * i < cols) row[col + 32 * i] = (uint8_t)((i < 4 ? lo : hi) >> 8 * (i % 4));
    }
}

// Sum (of one or two numbers), or largest of unsigned bits, over the threads that share a row: a CTA, or a part of one that has a
// barrier of its own (TEAMS).  `buffer`: 64 words of shared memory that nothing else uses until the next barrier but one.
template <int THREADS, int TEAMS> __device__ __forceinline__ void row_barrier() {
    if constexpr (TEAMS == 1) __syncthreads();
    else asm volatile("bar.sync %0, %1;" ::"r"(threadIdx.x / THREADS + 1), "n"(THREADS) : "memory");
}
template <int THREADS, int TEAMS, int N> __device__ __forceinline__ void row_sum(float (&v)[N], float *buffer) {
#pragma unroll
    for (int s = 16; s > 0; s /= 2)
#pragma unroll
        for (int n = 0; n < N; ++n) v[n] += __shfl_xor_sync(0xffffffffu, v[n], s);
    if constexpr (THREADS > 32) {
        const int lane = threadIdx.x & 31;
        if (lane == 0)
#pragma unroll
            for (int n = 0; n < N; ++n) buffer[n * 32 + threadIdx.x % THREADS / 32] = v[n];
        row_barrier<THREADS, TEAMS>();
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

// h w -> its 8-bit value before rounding, h w limit / most, where `most` is the largest |h w|.  The root cancels in this quotient, so
// it is often a tie of the rounding to 8 bits, and a unit's error decides which way that goes (5 of 100000 e4m3 values).  So the factor
// limit / most has two parts, which together are off by 2^-44 of it: quotients that 32 bits hold, as they do ties, come out exact (16.2 -> 17.2 us with scales of 128
// columns, 15.2 -> 15.3 with a scale a row).
struct Quotient {
    float high, low;
    __device__ __forceinline__ Pair operator()(Pair v) const { return fma(v, both(high), v * both(low)); }
    __device__ __forceinline__ float operator()(float v) const { return fmaf(v, high, v * low); }
};
// The scale, most r / limit with r what h w lacks of the norm, and that factor.  r is at most 1: where the scale is not zero, `most` is
// SMALLEST_MAX at least and the factor finite.  (most: the bits of a float, those of a NaN are above all others; reciprocal: of limit.)
__device__ __forceinline__ float make_scale(uint32_t most, float r, float limit, float reciprocal, Quotient &to) {
    const float m = __uint_as_float(most), y = m * r, q = y * reciprocal;
    float inverse; // off by one unit at most
    asm("rcp.approx.f32 %0, %1;" : "=f"(inverse) : "f"(m));
    const float high = inverse * limit, low = fmaf(-high, m, limit) * inverse;
    to.high = y < SMALLEST_MAX ? 0.f : y == y ? high : y;
    to.low = y < SMALLEST_MAX ? 0.f : low;
    // the quotient, with what is left of the division put back; an infinity stays one
    return y < SMALLEST_MAX ? 0.f : y < INFINITY ? fmaf(fmaf(-q, limit, y), reciprocal, q) : y;
}
// 1 / sqrt(v): one Newton step on the approximation
__device__ __forceinline__ float inverse_root(float v) {
    const float r = rsqrtf(v);
    return v < INFINITY ? fmaf(r * 0.5f, fmaf(-v * r, r, 1.f), r) : r;
}
// the power of two above the root of a row, and the root over it, 1/2 to 1 (a root of 0: 0; of a NaN: NaN)
__device__ __forceinline__ float power_of_two(float root, float &rest) {
    const uint32_t bits = __float_as_uint(root); // (never subnormal: the mean and epsilon are below 2^128)
    rest = __uint_as_float((bits & 0x007fffffu) | 0x3f000000u);
    return root > 0.f ? __uint_as_float((bits & 0x7f800000u) + 0x00800000u) : root;
}

__device__ __forceinline__ float largest(const Pair (&v)[4]) { // magnitude, or NaN
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float lo, hi;
        split(v[i], lo, hi);
        m = max_nan(max_nan(m, fabsf(lo)), fabsf(hi));
    }
    return m;
}

// The eight columns of a thread, 32 apart: a group is the same GROUP / 32 of them in all lanes (or one in half of them).  One group after
// the other: 4099 x 4096 bf16 that start anywhere, groups of 128, take 24 us instead of the 47 of all eight maxima at once, whose registers
// spill.  (That form also came out of ptxas 12.9 wrong at -O3, though not at -O1, once the quotient had more parts than one: in the kernels of
// four chunks every group had the first one's maximum.)
template <int GROUP>
__device__ __forceinline__ void scale_spread(float *scales, int col, int cols, float r, float limit, float reciprocal, float (&each)[8]) {
    constexpr int N = GROUP < 32 ? 1 : GROUP / 32;
#pragma unroll
    for (int k = 0; k < 8; k += N) {
        float m = 0.f;
#pragma unroll
        for (int i = k; i < k + N; ++i) m = max_nan(m, fabsf(each[i]));
        uint32_t most = __float_as_uint(m) & 0x7fffffffu;
        if constexpr (GROUP == 16) {
#pragma unroll
            for (int s = 1; s < 16; s *= 2) most = max(most, __shfl_xor_sync(0xffffffffu, most, s));
        } else {
            most = __reduce_max_sync(0xffffffffu, most);
        }
        Quotient to;
        const float s = make_scale(most, r, limit, reciprocal, to);
        if (col + 32 * k < cols && (col + 32 * k) % GROUP == 0) scales[(col + 32 * k) / GROUP] = s;
#pragma unroll
        for (int i = k; i < k + N; ++i) each[i] = to(each[i]);
    }
}

// h w to 8 bits by the scales of its groups, and the scales.  Groups of 16 to 256 columns, a power of two: in a warp's 256 columns
// they are whole lanes' (VEC), or one to eight times 32 columns of all lanes, or half of them.
template <bool VEC, int THREADS, int CHUNKS>
__device__ __forceinline__ void scale_groups(const NormArgs &a, float *scales, int thread, float r, float limit, float reciprocal, Pair (&v)[CHUNKS][4]) {
    const int shift = 31 - __clz(a.group), cols = (int)a.cols;
    if constexpr (VEC) {
        uint32_t m[CHUNKS];
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) m[c] = __float_as_uint(largest(v[c])) & 0x7fffffffu;
#pragma unroll
        for (int s = 1; s < 32; s *= 2)
            if (8 * s < a.group)
#pragma unroll
                for (int c = 0; c < CHUNKS; ++c) m[c] = max(m[c], __shfl_xor_sync(0xffffffffu, m[c], s));
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const int col = chunk_column<VEC>(c * THREADS + thread);
            Quotient to;
            const float s = make_scale(m[c], r, limit, reciprocal, to);
            if (col < cols && (col & (a.group - 1)) == 0) scales[col >> shift] = s;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[c][i] = to(v[c][i]);
        }
    } else {
        auto all = [&](auto spread) {
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c) {
                float each[8];
#pragma unroll
                for (int i = 0; i < 4; ++i) split(v[c][i], each[2 * i], each[2 * i + 1]);
                scale_spread<decltype(spread)::value>(scales, chunk_column<VEC>(c * THREADS + thread), cols, r, limit, reciprocal, each);
#pragma unroll
                for (int i = 0; i < 4; ++i) v[c][i] = pair(each[2 * i], each[2 * i + 1]);
            }
        };
        switch (a.group) {
            case 16: all(std::integral_constant<int, 16>()); break;
            case 32: all(std::integral_constant<int, 32>()); break;
            case 64: all(std::integral_constant<int, 64>()); break;
            case 128: all(std::integral_constant<int, 128>()); break;
            default: all(std::integral_constant<int, 256>());
        }
    }
}

template <typename D, bool VEC, int THREADS, int CHUNKS>
__device__ __forceinline__ void store_row(D *row, int thread, int cols, const Pair (&v)[CHUNKS][4]) {
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) Chunk<D, VEC>::store(row, chunk_column<VEC>(c * THREADS + thread), cols, v[c]);
}

// A CTA's threads, the rows that they work on at the same time, and the CTAs of an SM that registers are cut to.  (The gradient's
// CTAs have at least 256 threads, so that there are few parts of the weights' gradient.)
template <int THREADS> constexpr int BLOCK = THREADS == 32 ? 256 : THREADS;
template <int THREADS> constexpr int TEAMS = THREADS == 32 ? 8 : 1;
template <int THREADS> constexpr int BACKWARD_BLOCK = THREADS < 256 ? 256 : THREADS;
template <int THREADS> constexpr int BACKWARD_TEAMS = BACKWARD_BLOCK<THREADS> / THREADS;
template <typename T, bool VEC, int THREADS, int CHUNKS>
constexpr int FORWARD_CTAS = THREADS > 256 ? 1 : (VEC && sizeof(T) == 2 && CHUNKS <= 2 ? 768 : 512) / BLOCK<THREADS>;
template <int THREADS> constexpr int BACKWARD_CTAS = 512 / BACKWARD_BLOCK<THREADS>;
// whether registers hold a row that is on its way
template <typename T, bool VEC, int THREADS, int CHUNKS> constexpr bool FORWARD_AHEAD = CHUNKS <= 2 || (VEC && sizeof(T) == 2 && THREADS <= 256);
template <typename T, int CHUNKS> constexpr bool BACKWARD_AHEAD = CHUNKS * sizeof(T) <= 4;

// CTAs that stay take rows in turn; the next row is on its way while one is worked on, and the weights stay in registers.  (A CTA a
// row, nothing ahead: 8192 x 4096 41.8 us instead of 37.6.  Two rows ahead: 45, the copies between registers wait for the loads.)
template <typename T, bool VEC, int THREADS, int CHUNKS>
__global__ void __launch_bounds__(BLOCK<THREADS>, FORWARD_CTAS<T, VEC, THREADS, CHUNKS>) rms_norm_kernel(const __grid_constant__ NormArgs a) {
    __shared__ float sums[2][64];
    __shared__ uint32_t most[2][32];
    ptx::grid_dependency_wait();
    const int thread = threadIdx.x % THREADS, cols = (int)a.cols;
    const uint32_t step = gridDim.x * TEAMS<THREADS>, rows = (uint32_t)a.rows; // (below 2^31)
    uint32_t t = blockIdx.x * TEAMS<THREADS> + (THREADS == 32 ? threadIdx.x / 32 : 0);
    Chunk<T, VEC> x[CHUNKS], r[CHUNKS];
    auto load = [&](uint32_t row) {
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const int col = chunk_column<VEC>(c * THREADS + thread);
            x[c].load((const T *)a.src + row * a.src_ld, col, cols);
            if (a.residual) r[c].load((const T *)a.residual + row * a.residual_ld, col, cols);
        }
    };
    if (FORWARD_AHEAD<T, VEC, THREADS, CHUNKS> && t < rows) load(t);
    Pair w[CHUNKS][4];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) load_weights<T, VEC>(a, chunk_column<VEC>(c * THREADS + thread), w[c]);
    const float given = a.scaling == NORM_SCALE_GIVEN ? 1.f / ptx::ld_dependent(a.scales) : 1.f;
    const float limit = a.dst_dt == DT_S8 ? 127.f : 448.f, reciprocal = a.dst_dt == DT_S8 ? 1.f / 127.f : 1.f / 448.f;
    const float per_column = 1.f / (float)cols;
    for (int turn = 0; t < rows; t += step, turn ^= 1) {
        if (!FORWARD_AHEAD<T, VEC, THREADS, CHUNKS>) load(t);
        Pair h[CHUNKS][4], squares = both(0.f);
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            x[c].get(h[c]);
            if (a.residual) {
                Pair v[4];
                r[c].get(v);
#pragma unroll
                for (int i = 0; i < 4; ++i) h[c][i] = h[c][i] + v[i];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) squares = fma(h[c][i], h[c][i], squares);
        }
        if (FORWARD_AHEAD<T, VEC, THREADS, CHUNKS> && t + step < rows) load(t + step);
        if (a.sum) store_row<T, VEC, THREADS>((T *)a.sum + t * a.sum_ld, thread, cols, h);
        float sum[2];
        split(squares, sum[0], sum[1]);
        float total[1] = {sum[0] + sum[1]};
        row_sum<THREADS, 1>(total, sums[turn]);
        const float root = inverse_root(fmaf(total[0], per_column, a.epsilon));
        // The root before the weights: h is then below 2 sqrt(columns) (0 where the squares exceeded 32 bits), and its product with
        // the weight finite where the result is.  With made scales only a power of two of it, which leaves h as exact as it was; what
        // is left of the root goes into the scale.
        const bool made = a.scaling == NORM_SCALE_ROW || a.scaling == NORM_SCALE_GROUP;
        float rest;
        const Pair first = both(made ? power_of_two(root, rest) : root);
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) h[c][i] = h[c][i] * first * w[c][i];
        if (a.scaling == NORM_SCALE_ROW) {
            float m = 0.f;
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c) m = max_nan(m, largest(h[c]));
            Quotient to;
            const float s = make_scale(row_max<THREADS>(__float_as_uint(m) & 0x7fffffffu, most[turn]), rest, limit, reciprocal, to);
            if (thread == 0) a.scales[t] = s;
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) h[c][i] = to(h[c][i]);
        } else if (a.scaling == NORM_SCALE_GROUP) {
            scale_groups<VEC, THREADS>(a, a.scales + (int64_t)t * (cols / a.group), thread, rest, limit, reciprocal, h);
        } else if (a.scaling == NORM_SCALE_GIVEN) {
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) h[c][i] = h[c][i] * both(given);
        }
        switch (a.dst_dt) {
            case DT_F32: store_row<float, VEC, THREADS>((float *)a.dst + t * a.dst_ld, thread, cols, h); break;
            case DT_BF16: store_row<__nv_bfloat16, VEC, THREADS>((__nv_bfloat16 *)a.dst + t * a.dst_ld, thread, cols, h); break;
            case DT_F16: store_row<__half, VEC, THREADS>((__half *)a.dst + t * a.dst_ld, thread, cols, h); break;
            default: {
#pragma unroll
                for (int c = 0; c < CHUNKS; ++c) store_8bit<VEC>(a, t, chunk_column<VEC>(c * THREADS + thread), h[c]);
            }
        }
    }
}

// Gradient: CTAs that stay take rows in turn; the weights and this CTA's part of their gradient stay in registers, and the
// parts of all CTAs meet in the scratchpad, which the kernel behind this one adds up, in the same order every time.
template <typename T, bool VEC, int THREADS, int CHUNKS>
__global__ void __launch_bounds__(BACKWARD_BLOCK<THREADS>, BACKWARD_CTAS<THREADS>) rms_norm_backward_kernel(const __grid_constant__ NormArgs a) {
    constexpr int ROWS = BACKWARD_TEAMS<THREADS>;
    extern __shared__ __align__(16) float gathered[]; // several rows at a time: [ROWS][columns]
    __shared__ float sums[2][ROWS][64];
    ptx::grid_dependency_wait();
    const int thread = threadIdx.x % THREADS, team = threadIdx.x / THREADS, cols = (int)a.cols;
    const float per_column = 1.f / (float)cols;
    const uint32_t step = gridDim.x * ROWS, rows = (uint32_t)a.rows; // (below 2^31)
    uint32_t t = blockIdx.x * ROWS + team;
    Chunk<T, VEC> next_h[CHUNKS], next_dy[CHUNKS], next_more[CHUNKS];
    auto load = [&](uint32_t row) {
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const int col = chunk_column<VEC>(c * THREADS + thread);
            next_h[c].load((const T *)a.src + row * a.src_ld, col, cols);
            next_dy[c].load((const T *)a.diff_dst + row * a.diff_dst_ld, col, cols);
            if (a.residual) next_more[c].load((const T *)a.residual + row * a.residual_ld, col, cols);
        }
    };
    if (BACKWARD_AHEAD<T, CHUNKS> && t < rows) load(t);
    asm volatile("griddepcontrol.launch_dependents;"); // all CTAs are resident; what comes next waits for their end
    Pair w[CHUNKS][4], dw[CHUNKS][4];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
        load_weights<T, VEC>(a, chunk_column<VEC>(c * THREADS + thread), w[c]);
#pragma unroll
        for (int i = 0; i < 4; ++i) dw[c][i] = both(0.f);
    }
    for (int turn = 0; t < rows; t += step, turn ^= 1) {
        if (!BACKWARD_AHEAD<T, CHUNKS>) load(t);
        Chunk<T, VEC> h[CHUNKS], dy[CHUNKS], more[CHUNKS];
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            h[c] = next_h[c];
            dy[c] = next_dy[c];
            if (a.residual) more[c] = next_more[c];
        }
        if (BACKWARD_AHEAD<T, CHUNKS> && t + step < rows) load(t + step);
        Pair squares = both(0.f), products = both(0.f);
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            Pair x[4], g[4];
            h[c].get(x);
            dy[c].get(g);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                squares = fma(x[i], x[i], squares);
                products = fma(x[i] * w[c][i], g[i], products);
            }
        }
        float s[2], odd[2];
        split(squares, s[0], odd[0]);
        split(products, s[1], odd[1]);
        s[0] += odd[0];
        s[1] += odd[1];
        row_sum<THREADS, ROWS>(s, sums[turn][team]);
        const float r = inverse_root(fmaf(s[0], per_column, a.epsilon));
        // dh = r (z - h inner); where the squares exceeded 32 bits r is 0, and the products may have exceeded them too
        const Pair root = both(r), inner = both(r > 0.f ? -(s[1] * per_column * r * r) : 0.f);
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            Pair x[4], g[4], d[4];
            h[c].get(x);
            dy[c].get(g);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                d[i] = root * fma(g[i], w[c][i], x[i] * inner);
                dw[c][i] = fma(g[i], x[i] * root, dw[c][i]);
            }
            if (a.residual) {
                more[c].get(x);
#pragma unroll
                for (int i = 0; i < 4; ++i) d[i] = d[i] + x[i];
            }
            Chunk<T, VEC>::store((T *)a.diff_src + t * a.diff_src_ld, chunk_column<VEC>(c * THREADS + thread), cols, d);
        }
    }
    if (!a.parts) return;
    if constexpr (ROWS > 1) {
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) Chunk<float, VEC>::store(gathered + team * cols, chunk_column<VEC>(c * THREADS + thread), cols, dw[c]);
        __syncthreads();
        for (int col = threadIdx.x; col < cols; col += 256) {
            float sum = 0.f;
#pragma unroll
            for (int q = 0; q < ROWS; ++q) sum += gathered[q * cols + col];
            a.parts[blockIdx.x * a.cols + col] = sum;
        }
    } else {
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c)
            Chunk<float, VEC>::store(a.parts + blockIdx.x * a.cols, chunk_column<VEC>(c * THREADS + thread), cols, dw[c]);
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
        for (int p0 = warp; p0 < a.part_count; p0 += 8 * 32) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = p0 + 32 * i < a.part_count ? ptx::ld_dependent(a.parts + (p0 + 32 * i) * a.cols + col) : 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) sum += v[i];
        }
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

template <typename T, bool VEC, int THREADS, int CHUNKS> int launch_forward(const NormArgs &a, int sm_count, cudaStream_t st) {
    const int64_t ctas = (a.rows + TEAMS<THREADS> - 1) / TEAMS<THREADS>;
    return launch_dependent(rms_norm_kernel<T, VEC, THREADS, CHUNKS>, a,
            (unsigned)std::min<int64_t>(ctas, sm_count * FORWARD_CTAS<T, VEC, THREADS, CHUNKS>), BLOCK<THREADS>, 0, st);
}
template <typename T, bool VEC, int THREADS, int CHUNKS> int launch_backward(NormArgs &a, int sm_count, cudaStream_t st) {
    const int64_t ctas = (a.rows + BACKWARD_TEAMS<THREADS> - 1) / BACKWARD_TEAMS<THREADS>;
    // a part of the weights' gradient for each CTA: four rows at least, unless the SMs are too many
    a.part_count = (int)std::min<int64_t>(std::min<int64_t>(ctas, std::max<int64_t>(ctas / 4, sm_count)), sm_count * BACKWARD_CTAS<THREADS>);
    return launch_dependent(rms_norm_backward_kernel<T, VEC, THREADS, CHUNKS>, a, a.part_count, BACKWARD_BLOCK<THREADS>,
            BACKWARD_TEAMS<THREADS> > 1 ? BACKWARD_TEAMS<THREADS> * a.cols * sizeof(float) : 0, st);
}
// Threads of a row and its chunks of eight columns each: two chunks where a residual doubles what is in flight, four without one, which
// halves what is done once a thread (us with two / four: 8192 x 4096 with residual 37.7 / 39.2, 8192 x 1024 with 12.2 / 13.4; 4099 x 4096
// without, scales of 128 columns 17.6 / 17.2, one scale 13.0 / 13.2), and more where the row needs them.
template <typename T, bool VEC> int launch_form(NormArgs &a, bool backward, int sm_count, cudaStream_t st) {
    const int64_t chunks = VEC ? (a.cols + 7) / 8 : (a.cols + 255) / 256 * 32;
    if (backward) {
        if (chunks <= 32) return launch_backward<T, VEC, 32, 1>(a, sm_count, st);
        if (chunks <= 64) return launch_backward<T, VEC, 32, 2>(a, sm_count, st);
        if (chunks <= 128) return launch_backward<T, VEC, 64, 2>(a, sm_count, st);
        if (chunks <= 256) return launch_backward<T, VEC, 128, 2>(a, sm_count, st);
        if (chunks <= 512) return launch_backward<T, VEC, 256, 2>(a, sm_count, st);
        if (chunks <= 1024) return launch_backward<T, VEC, 512, 2>(a, sm_count, st);
        return launch_backward<T, VEC, 512, 4>(a, sm_count, st);
    }
    if (chunks <= 32) return launch_forward<T, VEC, 32, 1>(a, sm_count, st);
    if (chunks <= 64) return launch_forward<T, VEC, 32, 2>(a, sm_count, st);
    if constexpr (VEC && sizeof(T) == 2)
        if (!a.residual) {
            if (chunks <= 128) return launch_forward<T, VEC, 32, 4>(a, sm_count, st);
            if (chunks <= 256) return launch_forward<T, VEC, 64, 4>(a, sm_count, st);
            if (chunks <= 512) return launch_forward<T, VEC, 128, 4>(a, sm_count, st);
        }
    if (chunks <= 128) return launch_forward<T, VEC, 64, 2>(a, sm_count, st);
    if (chunks <= 256) return launch_forward<T, VEC, 128, 2>(a, sm_count, st);
    if (chunks <= 512) return launch_forward<T, VEC, 256, 2>(a, sm_count, st);
    if (chunks <= 768) return launch_forward<T, VEC, 256, 3>(a, sm_count, st);
    if (chunks <= 1024) return launch_forward<T, VEC, 256, 4>(a, sm_count, st);
    return launch_forward<T, VEC, 512, 4>(a, sm_count, st);
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

// a part of the weights' gradient for each CTA: two an SM at most
size_t norm_scratch_bytes(int64_t cols, int sm_count) { return (size_t)sm_count * 2 * cols * sizeof(float); }

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

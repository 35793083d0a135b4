// The experts' rows back to their tokens, and the gradient.
//   y[t]  = residual[t] + D(sum_j w[t,j] rows[position[t,j]])
//   drows[position[t,j]] = w[t,j] D(dy[t]),  dw[t,j] = <D(dy[t]), rows[position[t,j]]>
// D is dropout (or nothing).  A slot whose position is outside the rows (-1: its token went to no expert there) adds
// nothing, not even the product of its weight and an infinity, and its dw is zero.  Every row belongs to one slot, so the
// sums have one order and no atomics.  Bytes bound both: each row is read once (and written once, backward).
#include "launch.h"
#include "token_rows.cuh"

namespace qmm {

namespace {

constexpr int GROUP = 8; // rows of a token in flight at a time: their loads leave before the first is used

template <typename S, typename D, bool VEC, bool DROP>
__global__ void __launch_bounds__(256) combine_kernel(const __grid_constant__ CombineArgs a) {
    __shared__ __align__(16) uint32_t words[DROP && !VEC ? 8 * 128 : 4];
    ptx::grid_dependency_wait();
    constexpr int N = Cols<S, VEC>::N;
    const int64_t units = row_units<VEC>(a.cols, DROP), total = a.tokens * units;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= total) return; // (whole warps, where a warp works together)
    const int64_t t = total <= 0xffffffff ? (uint32_t)i / (uint32_t)units : i / units;
    const int64_t col = unit_column<VEC>(i - t * units, t, a.cols, DROP);
    Cols<D, VEC> res;
    if (a.residual) res.load((const D *)a.residual + t * a.residual_ld, col, a.cols);
    float acc[N];
#pragma unroll
    for (int n = 0; n < N; ++n) acc[n] = 0.f;
    const int *positions = a.positions + t * a.positions_ld;
    const float *weights = a.weights + t * a.weights_ld;
    for (int j0 = 0; j0 < a.choices; j0 += GROUP) {
        int pos[GROUP];
        float w[GROUP];
        Cols<S, VEC> x[GROUP];
#pragma unroll
        for (int j = 0; j < GROUP; ++j) {
            pos[j] = j0 + j < a.choices ? ptx::ld_dependent(positions + j0 + j) : -1;
            w[j] = a.weights && j0 + j < a.choices ? ptx::ld_dependent(weights + j0 + j) : 1.f;
        }
#pragma unroll
        for (int j = 0; j < GROUP; ++j)
            if ((uint32_t)pos[j] < (uint64_t)a.rows) x[j].load((const S *)a.src + (int64_t)pos[j] * a.cols, col, a.cols);
#pragma unroll
        for (int j = 0; j < GROUP; ++j)
            if ((uint32_t)pos[j] < (uint64_t)a.rows) {
                float v[N];
                x[j].get(v);
#pragma unroll
                for (int n = 0; n < N; ++n) acc[n] = fmaf(w[j], v[n], acc[n]);
            }
    }
    if constexpr (DROP) {
        const uint64_t seed = ld_dependent_u64(a.drop.seed), offset = ld_dependent_u64(a.drop.seed + 1);
        apply_dropout<VEC>(acc, a.drop, seed, offset, t, a.cols, col, words + (VEC ? 0 : threadIdx.x / 32 * 128));
    }
    if (a.residual) {
        float v[N];
        res.get(v);
#pragma unroll
        for (int n = 0; n < N; ++n) acc[n] += v[n];
    }
    Cols<D, VEC>::store((D *)a.dst + t * a.dst_ld, col, a.cols, acc);
}

// Zeros for the rows that belong to no slot, shared out over the grid.
template <typename S, bool VEC> __device__ __forceinline__ void zero_tail(const CombineArgs &a) {
    int64_t kept = ptx::ld_dependent(a.offsets + a.experts - 1);
    kept = kept < 0 ? 0 : kept > a.rows ? a.rows : kept;
    const int64_t end = a.rows * a.cols;
    S *p = (S *)a.diff_src;
    constexpr int STEP = VEC ? 16 / sizeof(S) : 1;
    for (int64_t i = kept * a.cols + ((int64_t)blockIdx.x * 256 + threadIdx.x) * STEP; i < end; i += (int64_t)gridDim.x * 256 * STEP) {
        if constexpr (VEC) *reinterpret_cast<uint4 *>(p + i) = make_uint4(0, 0, 0, 0);
        else p[i] = from_f32<S>(0.f);
    }
}

// THREADS of the 256 of a CTA work on a token: all of them, or a warp where rows are short.
template <typename S, typename D, bool VEC, bool DROP, int THREADS>
__global__ void __launch_bounds__(256) combine_backward_kernel(const __grid_constant__ CombineArgs a) {
    __shared__ __align__(16) uint32_t words[DROP && !VEC ? 8 * 128 : 4];
    __shared__ float partial[8][GROUP];
    ptx::grid_dependency_wait();
    constexpr int N = Cols<S, VEC>::N;
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    const int64_t t = THREADS == 256 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 8 + warp;
    const int64_t units = (row_units<VEC>(a.cols, DROP) + 31) / 32 * 32;
    if (t < a.tokens) {
        uint64_t seed = 0, offset = 0;
        if constexpr (DROP) {
            seed = ld_dependent_u64(a.drop.seed);
            offset = ld_dependent_u64(a.drop.seed + 1);
        }
        for (int j0 = 0; j0 < a.choices; j0 += GROUP) {
            int pos[GROUP];
            float w[GROUP], dot[GROUP];
#pragma unroll
            for (int j = 0; j < GROUP; ++j) {
                pos[j] = j0 + j < a.choices ? ptx::ld_dependent(a.positions + t * a.positions_ld + j0 + j) : -1;
                w[j] = j0 + j < a.choices ? ptx::ld_dependent(a.weights + t * a.weights_ld + j0 + j) : 0.f;
                dot[j] = 0.f;
            }
            for (int64_t u = threadIdx.x % THREADS; u < units; u += THREADS) {
                const int64_t col = unit_column<VEC>(u, t, a.cols, DROP);
                Cols<D, VEC> g;
                Cols<S, VEC> x[GROUP];
                g.load((const D *)a.diff_dst + t * a.diff_dst_ld, col, a.cols);
#pragma unroll
                for (int j = 0; j < GROUP; ++j)
                    if ((uint32_t)pos[j] < (uint64_t)a.rows) x[j].load((const S *)a.src + (int64_t)pos[j] * a.cols, col, a.cols);
                float dy[N];
                g.get(dy);
                if constexpr (DROP) apply_dropout<VEC>(dy, a.drop, seed, offset, t, a.cols, col, words + (VEC ? 0 : warp * 128));
#pragma unroll
                for (int j = 0; j < GROUP; ++j)
                    if ((uint32_t)pos[j] < (uint64_t)a.rows) {
                        float v[N], d[N];
                        x[j].get(v);
#pragma unroll
                        for (int n = 0; n < N; ++n) {
                            dot[j] = fmaf(dy[n], v[n], dot[j]);
                            d[n] = w[j] * dy[n];
                        }
                        Cols<S, VEC>::store((S *)a.diff_src + (int64_t)pos[j] * a.cols, col, a.cols, d);
                    }
            }
#pragma unroll
            for (int j = 0; j < GROUP; ++j)
#pragma unroll
                for (int s = 16; s > 0; s /= 2) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], s);
            if constexpr (THREADS == 256) {
                if (lane == 0)
#pragma unroll
                    for (int j = 0; j < GROUP; ++j) partial[warp][j] = dot[j];
                __syncthreads();
                if (threadIdx.x < GROUP && j0 + (int)threadIdx.x < a.choices) {
                    float sum = 0.f;
#pragma unroll
                    for (int q = 0; q < 8; ++q) sum += partial[q][threadIdx.x];
                    a.diff_weights[t * a.diff_weights_ld + j0 + threadIdx.x] = sum;
                }
                __syncthreads();
            } else if (lane == 0) {
#pragma unroll
                for (int j = 0; j < GROUP; ++j)
                    if (j0 + j < a.choices) a.diff_weights[t * a.diff_weights_ld + j0 + j] = dot[j];
            }
        }
    }
    zero_tail<S, VEC>(a);
}

template <typename S, typename D, bool DROP> int launch_forward(const CombineArgs &a, bool vec, cudaStream_t st) {
    const int64_t total = a.tokens * (vec ? row_units<true>(a.cols, DROP) : row_units<false>(a.cols, DROP));
    const int64_t grid = (total + 255) / 256;
    if (grid > 0x7fffffff) return 3;
    return launch_dependent(vec ? combine_kernel<S, D, true, DROP> : combine_kernel<S, D, false, DROP>, a, (unsigned)grid, 256, 0, st);
}

template <typename S, typename D, bool DROP> int launch_backward(const CombineArgs &a, bool vec, cudaStream_t st) {
    const int64_t units = vec ? row_units<true>(a.cols, DROP) : row_units<false>(a.cols, DROP);
    const bool wide = units > 64;
    const int64_t grid = wide ? a.tokens : (a.tokens + 7) / 8;
    if (grid > 0x7fffffff) return 3;
    void (*kernel)(CombineArgs) = vec ? (wide ? combine_backward_kernel<S, D, true, DROP, 256> : combine_backward_kernel<S, D, true, DROP, 32>)
                                      : (wide ? combine_backward_kernel<S, D, false, DROP, 256> : combine_backward_kernel<S, D, false, DROP, 32>);
    return launch_dependent(kernel, a, (unsigned)grid, 256, 0, st);
}

template <typename S, typename D> int launch_types(const CombineArgs &a, bool backward, cudaStream_t st) {
    const bool drop = a.drop.seed != nullptr;
    const int64_t ds = sizeof(D);
    bool vec = rows_aligned(a.src, a.cols * (int64_t)sizeof(S), a.rows) && (!drop || a.cols % 4 == 0 || a.tokens == 1);
    int rc;
    if (backward) {
        vec = vec && rows_aligned(a.diff_src, a.cols * (int64_t)sizeof(S), a.rows) && rows_aligned(a.diff_dst, a.diff_dst_ld * ds, a.tokens);
        rc = drop ? launch_backward<S, D, true>(a, vec, st) : launch_backward<S, D, false>(a, vec, st);
    } else {
        vec = vec && rows_aligned(a.dst, a.dst_ld * ds, a.tokens) && (!a.residual || rows_aligned(a.residual, a.residual_ld * ds, a.tokens));
        rc = drop ? launch_forward<S, D, true>(a, vec, st) : launch_forward<S, D, false>(a, vec, st);
    }
    if (rc == 0) count_launch();
    return rc;
}

template <typename S> int launch_dst(const CombineArgs &a, bool backward, cudaStream_t st) {
    switch (a.tok_dt) {
        case DT_F32: return launch_types<S, float>(a, backward, st);
        case DT_BF16: return launch_types<S, __nv_bfloat16>(a, backward, st);
        case DT_F16: return launch_types<S, __half>(a, backward, st);
        default: return 3;
    }
}

int launch_any(const CombineArgs &a, bool backward, cudaStream_t st) {
    switch (a.row_dt) {
        case DT_F32: return launch_dst<float>(a, backward, st);
        case DT_BF16: return launch_dst<__nv_bfloat16>(a, backward, st);
        case DT_F16: return launch_dst<__half>(a, backward, st);
        default: return 3;
    }
}

} // namespace

int launch_combine(const CombineArgs &a, cudaStream_t st) {
    if (a.tokens == 0 || a.cols == 0) return 0;
    return launch_any(a, false, st);
}

int launch_combine_backward(const CombineArgs &a, cudaStream_t st) {
    if (a.tokens == 0) return 0;
    return launch_any(a, true, st);
}

} // namespace qmm

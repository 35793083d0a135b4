// Dropout on the way into a residual stream: dst = residual + (kept ? src / (1 - p) : 0), with the mask made from a counter
// (token_rows.cuh) and never stored.  The gradient is the same operator on the gradient, without a residual: the same
// (seed, offset) makes the same mask.  Elementwise, so the floor is one read of src and residual and one write of dst.
#include "launch.h"
#include "token_rows.cuh"

namespace qmm {

namespace {

constexpr int SHARES = 2; // of a thread: their loads leave together, their generators run side by side

template <typename T, bool VEC, bool RES>
__global__ void __launch_bounds__(256) dropout_kernel(const __grid_constant__ DropoutArgs a) {
    __shared__ __align__(16) uint32_t shared_words[VEC ? 4 : 8 * 128];
    uint32_t *words = shared_words + (VEC ? 0 : threadIdx.x / 32 * 128);
    ptx::grid_dependency_wait();
    const int64_t units = row_units<VEC>(a.cols, true), total = a.rows * units;
    const int64_t first = (int64_t)blockIdx.x * (256 * SHARES) + threadIdx.x;
    int64_t t[SHARES], col[SHARES];
    bool on[SHARES]; // (whole warps, where a warp works together)
    Cols<T, VEC> x[SHARES], res[SHARES];
#pragma unroll
    for (int s = 0; s < SHARES; ++s) {
        const int64_t i = first + 256 * s;
        t[s] = a.rows == 1 ? 0 : total <= 0xffffffff ? (int64_t)((uint32_t)i / (uint32_t)units) : i / units;
        col[s] = unit_column<VEC>(i - t[s] * units, t[s], a.cols, true);
        on[s] = i < total;
        if (on[s]) {
            x[s].load((const T *)a.src + t[s] * a.src_ld, col[s], a.cols);
            if constexpr (RES) res[s].load((const T *)a.residual + t[s] * a.residual_ld, col[s], a.cols);
        }
    }
    const uint64_t seed = ld_dependent_u64(a.drop.seed), offset = ld_dependent_u64(a.drop.seed + 1);
    constexpr int N = Cols<T, VEC>::N;
    uint32_t u[SHARES][N];
#pragma unroll
    for (int s = 0; s < SHARES; ++s) random_words<VEC>(u[s], seed, offset, t[s], a.cols, col[s], words);
#pragma unroll
    for (int s = 0; s < SHARES; ++s) {
        if (!on[s]) continue;
        float v[N], r[N];
        x[s].get(v);
#pragma unroll
        for (int n = 0; n < N; ++n) v[n] = a.drop.drop_all ? 0.f : v[n] * a.drop.scale;
        drop(v, u[s], a.drop);
        if constexpr (RES) {
            res[s].get(r);
#pragma unroll
            for (int n = 0; n < N; ++n) v[n] += r[n];
        }
        Cols<T, VEC>::store((T *)a.dst + t[s] * a.dst_ld, col[s], a.cols, v);
    }
}

template <typename T> int launch_typed(const DropoutArgs &a, cudaStream_t st) {
    const bool vec = rows_aligned(a.src, a.src_ld * sizeof(T), a.rows) && rows_aligned(a.dst, a.dst_ld * sizeof(T), a.rows)
            && (!a.residual || rows_aligned(a.residual, a.residual_ld * sizeof(T), a.rows)) && (a.cols % 4 == 0 || a.rows == 1);
    const int64_t total = a.rows * (vec ? row_units<true>(a.cols, true) : row_units<false>(a.cols, true));
    const int64_t grid = (total + 256 * SHARES - 1) / (256 * SHARES);
    if (grid > 0x7fffffff) return 3;
    void (*kernel)(DropoutArgs) = vec ? (a.residual ? dropout_kernel<T, true, true> : dropout_kernel<T, true, false>)
                                      : (a.residual ? dropout_kernel<T, false, true> : dropout_kernel<T, false, false>);
    const int rc = launch_dependent(kernel, a, (unsigned)grid, 256, 0, st);
    if (rc == 0) count_launch();
    return rc;
}

} // namespace

int launch_dropout(const DropoutArgs &args, int sm_count, cudaStream_t st) {
    DropoutArgs a = args;
    if (a.rows == 0 || a.cols == 0) return 0;
    // dense tensors are one long row, whatever the width
    if (a.src_ld == a.cols && a.dst_ld == a.cols && (!a.residual || a.residual_ld == a.cols)) {
        a.cols *= a.rows;
        a.rows = 1;
    }
    switch (a.dt) {
        case DT_F32: return launch_typed<float>(a, st);
        case DT_BF16: return launch_typed<__nv_bfloat16>(a, st);
        case DT_F16: return launch_typed<__half>(a, st);
        default: return 3;
    }
}

} // namespace qmm

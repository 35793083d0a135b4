// Dropout on the way into a residual stream: dst = residual + (kept ? src / (1 - p) : 0), with the mask made from a counter
// (token_rows.cuh) and never stored.  The gradient is the same operator on the gradient, without a residual: the same
// (seed, offset) makes the same mask.
//
// The floor is one read of src and residual and one write of dst; beside it stands the generator, whose 20 wide products a
// block of four elements leave the SM at 32 a clock: 19 us for 8192 x 4096 elements, whatever their type.  Both run side by
// side as long as nothing else fills the issue slots, so the usual form - dense tensors, one long row - computes one address
// a tensor and keeps or drops with one comparison and one predicated multiply-add.
#include <algorithm>
#include <type_traits>

#include "launch.h"
#include "token_rows.cuh"

namespace qmm {

namespace {

__device__ __forceinline__ float keep_add(uint32_t u, const DropoutState &d, float v, float residual) {
    return u >= d.threshold ? fmaf(v, d.scale, residual) : residual;
}

// Rows that start on 16-byte boundaries, and on multiples of four elements: eight neighbouring columns a share, two shares a
// thread at a time.  The loads leave before the generator runs, which takes longer than they do.  Where 16-bit elements leave
// the generator in front, the grid stays, four CTAs an SM; 32-bit elements wait for memory, and more CTAs on their way bring it
// sooner.  8192 x 4096, the same inputs every call, us gone / staying: bf16 31.7 / 31.1, with residual 32.5 / 32.5 (five CTAs
// 33.7, one share 35.7); f32 40.5 / 54.2, with residual 59.0 / 68.9.
constexpr int SHARES = 2;
constexpr int CTAS = 4;

constexpr int SPREAD = 256 * 8, PIECE = SPREAD * SHARES; // columns from share to share of a thread; of a CTA at a time

// Dense tensors: one row.
template <typename T, bool RES, bool WHOLE>
__device__ __forceinline__ void drop_piece(const DropoutArgs &a, uint64_t seed, uint64_t offset, const T *src, const T *residual, T *dst,
        int64_t col, uint64_t block) {
    Cols<T, true> x[SHARES], res[SHARES];
    const int64_t end = WHOLE ? INT64_MAX : a.cols;
#pragma unroll
    for (int s = 0; s < SHARES; ++s)
        if (WHOLE || col + SPREAD * s < end) {
            x[s].load_ragged(src + SPREAD * s, WHOLE ? 8 : end - col - SPREAD * s);
            if constexpr (RES) res[s].load_ragged(residual + SPREAD * s, WHOLE ? 8 : end - col - SPREAD * s);
        }
    uint32_t u[SHARES][8];
#pragma unroll
    for (int s = 0; s < SHARES; ++s)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint4 r = philox(seed, offset, block + SPREAD / 4 * s + h);
            u[s][4 * h] = r.x; u[s][4 * h + 1] = r.y; u[s][4 * h + 2] = r.z; u[s][4 * h + 3] = r.w;
        }
#pragma unroll
    for (int s = 0; s < SHARES; ++s)
        if (WHOLE || col + SPREAD * s < end) {
            float v[8], r[8];
            x[s].get(v);
            if constexpr (RES) res[s].get(r);
#pragma unroll
            for (int n = 0; n < 8; ++n) v[n] = keep_add(u[s][n], a.drop, v[n], RES ? r[n] : 0.f);
            Cols<T, true>::store_ragged(dst + SPREAD * s, WHOLE ? 8 : end - col - SPREAD * s, v);
        }
}

// A thread's shares begin at src[s], with left[s] columns of the row from there (WHOLE: eight at least).
template <typename T, bool RES, bool WHOLE>
__device__ __forceinline__ void drop_shares(const DropoutArgs &a, uint64_t seed, uint64_t offset, const T *const (&src)[SHARES],
        const T *const (&residual)[SHARES], T *const (&dst)[SHARES], const int64_t (&left)[SHARES], const uint64_t (&block)[SHARES]) {
    Cols<T, true> x[SHARES], res[SHARES];
#pragma unroll
    for (int s = 0; s < SHARES; ++s)
        if (WHOLE || left[s] > 0) {
            x[s].load_ragged(src[s], WHOLE ? 8 : left[s]);
            if constexpr (RES) res[s].load_ragged(residual[s], WHOLE ? 8 : left[s]);
        }
    uint32_t u[SHARES][8];
#pragma unroll
    for (int s = 0; s < SHARES; ++s)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint4 r = philox(seed, offset, block[s] + h);
            u[s][4 * h] = r.x; u[s][4 * h + 1] = r.y; u[s][4 * h + 2] = r.z; u[s][4 * h + 3] = r.w;
        }
#pragma unroll
    for (int s = 0; s < SHARES; ++s)
        if (WHOLE || left[s] > 0) {
            float v[8], r[8];
            x[s].get(v);
            if constexpr (RES) res[s].get(r);
#pragma unroll
            for (int n = 0; n < 8; ++n) v[n] = keep_add(u[s][n], a.drop, v[n], RES ? r[n] : 0.f);
            Cols<T, true>::store_ragged(dst[s], WHOLE ? 8 : left[s], v);
        }
}

// One row.
template <typename T, bool RES> __global__ void __launch_bounds__(256, CTAS) dropout_dense_kernel(const __grid_constant__ DropoutArgs a) {
    ptx::grid_dependency_wait();
    const uint64_t seed = same_in_warp(ld_dependent_u64(a.drop.seed)), offset = ld_dependent_u64(a.drop.seed + 1);
    const int64_t step = (int64_t)gridDim.x * PIECE;
    int64_t col = (int64_t)blockIdx.x * PIECE + threadIdx.x * 8;
    const T *src = (const T *)a.src + col, *residual = RES ? (const T *)a.residual + col : nullptr;
    T *dst = (T *)a.dst + col;
    int64_t left = a.cols - (int64_t)blockIdx.x * PIECE; // from the piece's beginning
    for (; left >= PIECE; left -= step) {
        drop_piece<T, RES, true>(a, seed, offset, src, residual, dst, 0, (uint64_t)col >> 2);
        col += step;
        src += step;
        if constexpr (RES) residual += step;
        dst += step;
    }
    if (left > 0) drop_piece<T, RES, false>(a, seed, offset, src, residual, dst, col, (uint64_t)col >> 2);
}

// Several rows: shares are counted over all of them, and each finds its own.
template <typename T, bool RES> __global__ void __launch_bounds__(256, CTAS) dropout_rows_kernel(const __grid_constant__ DropoutArgs a) {
    ptx::grid_dependency_wait();
    const uint64_t seed = same_in_warp(ld_dependent_u64(a.drop.seed)), offset = ld_dependent_u64(a.drop.seed + 1);
    const int64_t units = (a.cols + 7) / 8, total = a.rows * units;
    for (int64_t first = (int64_t)blockIdx.x * (256 * SHARES); first < total; first += (int64_t)gridDim.x * (256 * SHARES)) {
        const T *src[SHARES], *residual[SHARES];
        T *dst[SHARES];
        int64_t left[SHARES];
        uint64_t block[SHARES];
#pragma unroll
        for (int s = 0; s < SHARES; ++s) {
            const int64_t i = first + threadIdx.x + 256 * s;
            const int64_t t = total <= 0xffffffff ? (int64_t)((uint32_t)i / (uint32_t)units) : i / units, col = (i - t * units) * 8;
            src[s] = (const T *)a.src + t * a.src_ld + col;
            residual[s] = (const T *)a.residual + t * a.residual_ld + col;
            dst[s] = (T *)a.dst + t * a.dst_ld + col;
            left[s] = i < total ? a.cols - col : 0;
            block[s] = (uint64_t)(t * a.cols + col) >> 2;
        }
        if (a.cols % 8 == 0 && first + 256 * SHARES <= total) drop_shares<T, RES, true>(a, seed, offset, src, residual, dst, left, block);
        else drop_shares<T, RES, false>(a, seed, offset, src, residual, dst, left, block);
    }
}

// Rows that start anywhere: a warp takes 256 columns, 32 beside one another at a time, so that its accesses stay contiguous;
// the 256 begin at a multiple of four elements of the whole tensor, up to three columns before the row, and the words of
// their 64 blocks go through shared memory to the lanes that need them.
constexpr int SPAN = 256;

template <typename T, bool RES> __global__ void __launch_bounds__(256) dropout_any_kernel(const __grid_constant__ DropoutArgs a) {
    __shared__ __align__(16) uint32_t shared_words[8 * SPAN];
    ptx::grid_dependency_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    uint32_t *words = shared_words + warp * SPAN;
    const uint64_t seed = same_in_warp(ld_dependent_u64(a.drop.seed)), offset = ld_dependent_u64(a.drop.seed + 1);
    const int64_t spans = (a.cols + 3 + SPAN - 1) / SPAN, total = a.rows * spans;
    for (int64_t item = (int64_t)blockIdx.x * 8 + warp; item < total; item += (int64_t)gridDim.x * 8) {
        const int64_t t = total <= 0xffffffff ? (int64_t)((uint32_t)item / (uint32_t)spans) : item / spans;
        const int64_t start = t * a.cols, begin = (item - t * spans) * SPAN - (start & 3); // the span's first column
        const T *src = (const T *)a.src + t * a.src_ld + begin, *residual = (const T *)a.residual + t * a.residual_ld + begin;
        T *dst = (T *)a.dst + t * a.dst_ld + begin;
        // columns of the span that are there: [low, high)
        const int low = begin < 0 ? (int)-begin : 0, high = (int)min((int64_t)SPAN, a.cols - begin);
        const uint64_t block = (uint64_t)(start + begin) >> 2;
        auto span = [&](auto whole) {
            T x[SPAN / 32], res[SPAN / 32];
#pragma unroll
            for (int i = 0; i < SPAN / 32; ++i) {
                const int c = 32 * i + lane;
                if (whole || (c >= low && c < high)) {
                    x[i] = src[c];
                    if constexpr (RES) res[i] = residual[c];
                }
            }
            __syncwarp();
            reinterpret_cast<uint4 *>(words)[lane] = philox(seed, offset, block + lane);
            reinterpret_cast<uint4 *>(words)[lane + 32] = philox(seed, offset, block + lane + 32);
            __syncwarp();
#pragma unroll
            for (int i = 0; i < SPAN / 32; ++i) {
                const int c = 32 * i + lane;
                if (whole || (c >= low && c < high)) dst[c] = from_f32<T>(keep_add(words[c], a.drop, to_f32(x[i]), RES ? to_f32(res[i]) : 0.f));
            }
        };
        if (low == 0 && high == SPAN) span(std::true_type());
        else span(std::false_type());
    }
}

// p = 1: nothing is kept, and no comparison with a 32-bit word says so
template <typename T> __global__ void __launch_bounds__(256) dropout_all_kernel(const __grid_constant__ DropoutArgs a) {
    ptx::grid_dependency_wait();
    const int64_t total = a.rows * a.cols;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t t = i / a.cols, c = i - t * a.cols;
        ((T *)a.dst)[t * a.dst_ld + c] = a.residual ? ((const T *)a.residual)[t * a.residual_ld + c] : from_f32<T>(0.f);
    }
}

template <typename T> int launch_typed(const DropoutArgs &a, int sm_count, cudaStream_t st) {
    const bool vec = rows_aligned(a.src, a.src_ld * sizeof(T), a.rows) && rows_aligned(a.dst, a.dst_ld * sizeof(T), a.rows)
            && (!a.residual || rows_aligned(a.residual, a.residual_ld * sizeof(T), a.rows)) && (a.cols % 4 == 0 || a.rows == 1);
    void (*kernel)(DropoutArgs);
    int64_t grid;
    if (a.drop.drop_all) {
        kernel = dropout_all_kernel<T>;
        grid = std::min<int64_t>((a.rows * a.cols + 255) / 256, (int64_t)sm_count * 16);
    } else if (vec) {
        kernel = a.rows == 1 ? (a.residual ? dropout_dense_kernel<T, true> : dropout_dense_kernel<T, false>)
                             : (a.residual ? dropout_rows_kernel<T, true> : dropout_rows_kernel<T, false>);
        grid = (a.rows * ((a.cols + 7) / 8) + 256 * SHARES - 1) / (256 * SHARES);
        if (sizeof(T) == 2) grid = std::min(grid, (int64_t)sm_count * CTAS);
    } else {
        kernel = a.residual ? dropout_any_kernel<T, true> : dropout_any_kernel<T, false>;
        grid = std::min((a.rows * ((a.cols + 3 + SPAN - 1) / SPAN) + 7) / 8, (int64_t)sm_count * 6);
    }
    if (grid > 0x7fffffff) return 3;
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
        case DT_F32: return launch_typed<float>(a, sm_count, st);
        case DT_BF16: return launch_typed<__nv_bfloat16>(a, sm_count, st);
        case DT_F16: return launch_typed<__half>(a, sm_count, st);
        default: return 3;
    }
}

} // namespace qmm

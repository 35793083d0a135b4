// The experts' rows back to their tokens, and the gradient.
//   y[t]  = residual[t] + D(sum_j w[t,j] rows[position[t,j]])
//   drows[position[t,j]] = w[t,j] D(dy[t]),  dw[t,j] = <D(dy[t]), rows[position[t,j]]>
// D is dropout (or nothing).  A slot whose position is outside the rows (-1: its token went to no expert there) adds
// nothing, not even the product of its weight and an infinity, and its dw is zero.  Every row belongs to one slot, so the
// sums have one order and no atomics.  Bytes bound both: each row is read once (and written once, backward).
#include <algorithm>

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

// acc[0..1] += w * v[0..1], both in one instruction
__device__ __forceinline__ void fma2(float &a0, float &a1, float w, float v0, float v1) {
    asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %2};\n\tmov.b64 b, {%3, %4};\n\tmov.b64 c, {%0, %1};\n\t"
        "fma.rn.f32x2 c, a, b, c;\n\tmov.b64 {%0, %1}, c;\n\t}"
        : "+f"(a0), "+f"(a1) : "f"(w), "f"(v0), "f"(v1));
}

// The same sum for many tokens: one CTA per SM, whose first warp streams the rows' segments through a ring of stages in
// shared memory with bulk copies - as many bytes in flight as the ring holds, whatever the other warps do - and whose
// others sum them.  An item is a segment of up to 2048 columns of one token, a stage its rows' segments.
constexpr int BULK_WARPS = 8; // that sum an item: 8 columns a thread
constexpr int BULK_GROUPS = 3; // of such warps, which take the items in turn
constexpr int BULK_THREADS = 32 + BULK_GROUPS * BULK_WARPS * 32;
constexpr int BULK_COLS = BULK_WARPS * 32 * 8;
constexpr int BULK_MAX_STAGES = 16;
constexpr int BULK_RING = 200 * 1024;

struct BulkPlan {
    CombineArgs a;
    int segment; // columns of an item
    int stages;
};

template <typename S, typename D, bool DROP>
__global__ void __launch_bounds__(BULK_THREADS, 1) combine_bulk_kernel(const __grid_constant__ BulkPlan p) {
    extern __shared__ __align__(128) char ring[];
    __shared__ uint64_t full[BULK_MAX_STAGES], empty[BULK_MAX_STAGES];
    __shared__ int late; // a wait ran out
    const CombineArgs &a = p.a;
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    if (threadIdx.x == 0) {
        late = 0;
        for (int s = 0; s < p.stages; ++s) {
            ptx::mbar_init(&full[s], 1);
            ptx::mbar_init(&empty[s], BULK_WARPS);
        }
        ptx::fence_barrier_init();
    }
    __syncthreads();
    ptx::grid_dependency_wait();
    const uint32_t segments = (uint32_t)((a.cols + p.segment - 1) / p.segment);
    const int64_t items = a.tokens * segments;
    const int row_bytes = p.segment * (int)sizeof(S), stage_bytes = a.choices * row_bytes;
    auto token_of = [&](int64_t i) { return items <= 0xffffffff ? (int64_t)((uint32_t)i / segments) : i / segments; };
    // lane j: position (and weight) of choice j, fetched an item ahead
    auto position = [&](int64_t t) { return lane < a.choices ? ptx::ld_dependent(a.positions + t * a.positions_ld + lane) : -1; };
    auto weight = [&](int64_t t) { return lane < a.choices && a.weights ? ptx::ld_dependent(a.weights + t * a.weights_ld + lane) : 1.f; };
    int64_t item = blockIdx.x;
    int stage = 0;
    uint32_t phase = 0;
    bool failed = false;
    if (warp == 0) {
        int pos = item < items ? position(token_of(item)) : -1;
        for (; item < items; item += gridDim.x) {
            const int64_t next = item + gridDim.x, t = token_of(item);
            const int next_pos = next < items ? position(token_of(next)) : -1;
            const int64_t col = (item - t * segments) * p.segment;
            const uint32_t bytes = (uint32_t)min((int64_t)p.segment, a.cols - col) * (uint32_t)sizeof(S);
            const bool there = (uint32_t)pos < a.rows;
            if (!__all_sync(0xffffffffu, ptx::mbar_wait(&empty[stage], phase ^ 1))) {
                failed = true;
                break;
            }
            const uint32_t rows = __popc(__ballot_sync(0xffffffffu, there));
            if (lane == 0) ptx::mbar_arrive_expect_tx(&full[stage], rows * bytes);
            __syncwarp();
            if (there) ptx::bulk_load(ring + stage * stage_bytes + lane * row_bytes, (const S *)a.src + (int64_t)pos * a.cols + col, bytes, &full[stage]);
            pos = next_pos;
            if (++stage == p.stages) {
                stage = 0;
                phase ^= 1;
            }
        }
    } else {
        uint64_t seed = 0, offset = 0;
        if constexpr (DROP) {
            seed = ld_dependent_u64(a.drop.seed);
            offset = ld_dependent_u64(a.drop.seed + 1);
        }
        const int group = (warp - 1) / BULK_WARPS;
        const int mine = ((warp - 1) % BULK_WARPS * 32 + lane) * 8; // first column within the segment
        const bool active = mine < p.segment;
        auto column = [&](int64_t i, int64_t t) { return (i - t * segments) * p.segment + mine; };
        Cols<D, true> res, next_res;
        int64_t t = 0, tn = 0;
        int pos = -1;
        float w = 1.f;
        const int64_t step = (int64_t)gridDim.x * BULK_GROUPS;
        item += (int64_t)gridDim.x * group;
        stage = group;
        while (stage >= p.stages) {
            stage -= p.stages;
            phase ^= 1;
        }
        if (item < items) {
            t = token_of(item);
            pos = position(t);
            w = weight(t);
            if (a.residual && active) res.load((const D *)a.residual + t * a.residual_ld, column(item, t), a.cols);
        }
        for (; item < items; item += step) {
            const int64_t next = item + step, col = column(item, t);
            int next_pos = -1;
            float next_w = 1.f;
            if (next < items) {
                tn = token_of(next);
                next_pos = position(tn);
                next_w = weight(tn);
                if (a.residual && active) next_res.load((const D *)a.residual + tn * a.residual_ld, column(next, tn), a.cols);
            }
            const uint32_t there = __ballot_sync(0xffffffffu, (uint32_t)pos < a.rows);
            float acc[8];
#pragma unroll
            for (int n = 0; n < 8; ++n) acc[n] = 0.f;
            if (!__all_sync(0xffffffffu, ptx::mbar_wait(&full[stage], phase))) {
                failed = true;
                break;
            }
            const S *rows = (const S *)(ring + stage * stage_bytes) + mine;
            for (int j0 = 0; j0 < a.choices; j0 += GROUP) {
#pragma unroll
                for (int j = 0; j < GROUP; ++j) {
                    const float wj = __shfl_sync(0xffffffffu, w, (j0 + j) & 31);
                    if (j0 + j < 32 && (there >> (j0 + j)) & 1) {
                        Cols<S, true> x;
                        if (active) x.load_shared(rows + (j0 + j) * p.segment);
                        float v[8];
                        x.get(v);
#pragma unroll
                        for (int n = 0; n < 8; n += 2) fma2(acc[n], acc[n + 1], wj, v[n], v[n + 1]);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(&empty[stage]);
            if (active && col < a.cols) {
                if constexpr (DROP) apply_dropout<true>(acc, a.drop, seed, offset, t, a.cols, col, nullptr);
                if (a.residual) {
                    float v[8];
                    res.get(v);
#pragma unroll
                    for (int n = 0; n < 8; ++n) acc[n] += v[n];
                }
                Cols<D, true>::store((D *)a.dst + t * a.dst_ld, col, a.cols, acc);
            }
            t = tn;
            pos = next_pos;
            w = next_w;
            res = next_res;
            stage += BULK_GROUPS;
            while (stage >= p.stages) {
                stage -= p.stages;
                phase ^= 1;
            }
        }
    }
    if (failed) late = 1;
    __syncthreads();
    if (late && threadIdx.x == 0) {
        // copies may still be on their way to warps that gave up: every stage's last phase ends before the memory goes
        for (int s = 0; s < p.stages; ++s)
            for (int parity = 0; parity < 2; ++parity) (void)ptx::mbar_wait(&full[s], parity, 500000000ull);
        if (a.status) atomicExch(a.status, 5);
    }
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

template <typename S, typename D, bool DROP> int launch_bulk(const CombineArgs &a, int sm_count, cudaStream_t st) {
    BulkPlan p {};
    p.a = a;
    // stages of at least four to the ring, segments of whole warps' shares
    const int most = BULK_RING / 4 / (a.choices * (int)sizeof(S)) / 256 * 256;
    const int wide = (int)std::min<int64_t>(BULK_COLS, (a.cols + 255) / 256 * 256);
    p.segment = std::max(256, std::min(most, wide));
    p.stages = std::min(BULK_MAX_STAGES, BULK_RING / (a.choices * p.segment * (int)sizeof(S)));
    const int64_t items = a.tokens * ((a.cols + p.segment - 1) / p.segment);
    static std::atomic<unsigned long long> done;
    if (!opt_in_dynamic_smem(combine_bulk_kernel<S, D, DROP>, BULK_RING, done)) return 5;
    return launch_dependent(combine_bulk_kernel<S, D, DROP>, p, (unsigned)std::min<int64_t>(items, sm_count), BULK_THREADS, BULK_RING, st);
}

template <typename S, typename D, bool DROP> int launch_forward(const CombineArgs &a, bool vec, int sm_count, cudaStream_t st) {
    const int64_t total = a.tokens * (vec ? row_units<true>(a.cols, DROP) : row_units<false>(a.cols, DROP));
    const int64_t grid = (total + 255) / 256;
    if (vec && a.cols * (int64_t)sizeof(S) % 16 == 0 && a.cols * (int64_t)sizeof(S) >= 1024 && a.tokens >= 4 * sm_count)
        return launch_bulk<S, D, DROP>(a, sm_count, st);
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

template <typename S, typename D> int launch_types(const CombineArgs &a, bool backward, int sm_count, cudaStream_t st) {
    const bool drop = a.drop.seed != nullptr;
    const int64_t ds = sizeof(D);
    bool vec = rows_aligned(a.src, a.cols * (int64_t)sizeof(S), a.rows) && (!drop || a.cols % 4 == 0 || a.tokens == 1);
    int rc;
    if (backward) {
        vec = vec && rows_aligned(a.diff_src, a.cols * (int64_t)sizeof(S), a.rows) && rows_aligned(a.diff_dst, a.diff_dst_ld * ds, a.tokens);
        rc = drop ? launch_backward<S, D, true>(a, vec, st) : launch_backward<S, D, false>(a, vec, st);
    } else {
        vec = vec && rows_aligned(a.dst, a.dst_ld * ds, a.tokens) && (!a.residual || rows_aligned(a.residual, a.residual_ld * ds, a.tokens));
        rc = drop ? launch_forward<S, D, true>(a, vec, sm_count, st) : launch_forward<S, D, false>(a, vec, sm_count, st);
    }
    if (rc == 0) count_launch();
    return rc;
}

template <typename S> int launch_dst(const CombineArgs &a, bool backward, int sm_count, cudaStream_t st) {
    switch (a.tok_dt) {
        case DT_F32: return launch_types<S, float>(a, backward, sm_count, st);
        case DT_BF16: return launch_types<S, __nv_bfloat16>(a, backward, sm_count, st);
        case DT_F16: return launch_types<S, __half>(a, backward, sm_count, st);
        default: return 3;
    }
}

int launch_any(const CombineArgs &a, bool backward, int sm_count, cudaStream_t st) {
    switch (a.row_dt) {
        case DT_F32: return launch_dst<float>(a, backward, sm_count, st);
        case DT_BF16: return launch_dst<__nv_bfloat16>(a, backward, sm_count, st);
        case DT_F16: return launch_dst<__half>(a, backward, sm_count, st);
        default: return 3;
    }
}

} // namespace

int launch_combine(const CombineArgs &a, int sm_count, cudaStream_t st) {
    if (a.tokens == 0 || a.cols == 0) return 0;
    return launch_any(a, false, sm_count, st);
}

int launch_combine_backward(const CombineArgs &a, int sm_count, cudaStream_t st) {
    if (a.tokens == 0) return 0;
    return launch_any(a, true, sm_count, st);
}

} // namespace qmm

// The experts' rows back to their tokens, and the gradient.
//   y[t]  = residual[t] + D(sum_j w[t,j] rows[position[t,j]])
//   drows[position[t,j]] = w[t,j] D(dy[t]),  dw[t,j] = <D(dy[t]), rows[position[t,j]]>
// D is dropout (or nothing).  A slot whose position is outside the groups' rows (-1: its token went to no expert there; at
// or behind the last offset) adds nothing, not even the product of its weight and an infinity, and its dw is zero.  Every row
// belongs to one slot, so the sums have one order and no atomics.  Bytes bound both: each row is read once (and written once,
// backward).
#include <algorithm>

#include "launch.h"
#include "token_rows.cuh"

namespace qmm {

namespace {

// Rows that the groups hold.  What lies behind is nobody's: forward does not read it, backward zeroes it in one place.
__device__ __forceinline__ uint32_t rows_of_groups(const CombineArgs &a) {
    const int last = ptx::ld_dependent(a.offsets + a.experts - 1);
    return last < 0 ? 0u : (uint32_t)min((int64_t)last, a.rows);
}

// GROUP rows of a token are in flight at a time: their loads leave before the first is used.  As many as a token has, up to
// eight: what eight take in registers costs a token of fewer rows its warps (when the gradient was given its groups, 4096 x 4096
// bf16: two rows 55 us in groups of eight / 34 of two, four rows 72 in groups of eight / 56 of four).

template <typename S, typename D, bool VEC, bool DROP, int GROUP>
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
        // (read here and not before the loop: held over it, the bound takes 10 registers and a CTA an SM where rows start anywhere,
        // 3000 x 8 x 2047 bf16 with dropout 47 us this way / 86)
        const uint32_t kept = rows_of_groups(a);
#pragma unroll
        for (int j = 0; j < GROUP; ++j) pos[j] = (uint32_t)pos[j] < kept ? pos[j] : -1;
#pragma unroll
        for (int j = 0; j < GROUP; ++j)
            if (pos[j] >= 0) x[j].load((const S *)a.src + (int64_t)pos[j] * a.cols, col, a.cols);
#pragma unroll
        for (int j = 0; j < GROUP; ++j)
            if (pos[j] >= 0) {
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

// The same sum for many tokens: one CTA per SM, whose first warps stream rows (and residuals) through a ring of stages in
// shared memory with bulk copies - as many bytes in flight as the ring holds, whatever the other warps do - and whose
// others sum them.  An item fills a stage: a segment of up to 2048 columns of one token, or several tokens whose rows are
// shorter.  A group of four warps works on an item, 16 columns a thread; the groups take the items in turn.
// Three warps issue the copies: one takes about 0.4 us an item and 0.04 us a row, which held 8192 tokens x 8 rows x 4096 bf16
// with dropout at 116 us and 4096 x 8 x 512 at 14.6 (three: 101 and 9.0; four: no better).
constexpr int BULK_WARPS = 4, BULK_GROUPS = 6;
constexpr int PRODUCERS = 3;
constexpr int BULK_THREADS = (PRODUCERS + BULK_GROUPS * BULK_WARPS) * 32;
constexpr int WARP_COLS = 512;
constexpr int BULK_MAX_STAGES = 24;
constexpr int BULK_RING = 208 * 1024;

struct BulkPlan {
    CombineArgs a;
    int warps; // of a token's segment
    uint32_t segments; // of a token's columns
    uint32_t items;
    int tokens; // of an item
    int stride; // elements from row to row of a stage
    int residuals; // bytes from a stage's beginning to its residuals
    int stage_bytes;
    int stages; // a multiple of the groups: a stage always serves the same group
    int groups; // at work
};

template <typename S, typename D, bool DROP>
__global__ void __launch_bounds__(BULK_THREADS, 1) combine_bulk_kernel(const __grid_constant__ BulkPlan p) {
    extern __shared__ __align__(128) char ring[];
    __shared__ uint64_t full[BULK_MAX_STAGES], empty[BULK_MAX_STAGES];
    __shared__ float weights[BULK_MAX_STAGES][32]; // of an item's rows
    __shared__ uint32_t present[BULK_MAX_STAGES]; // its rows that are there
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
    const uint32_t segments = p.segments, items = p.items;
    const int segment = p.warps * WARP_COLS;
    bool failed = false;
    if (warp < PRODUCERS) {
        // Serves every PRODUCERS-th group, in the order of their items.  A lane holds position and weight of a row; as many
        // items as have lanes are fetched together, two batches ahead.
        const int k = a.choices, rows = p.tokens * k, batch = 32 / rows;
        const uint32_t kept = rows_of_groups(a);
        const int of = lane / rows, row = lane - of * rows; // the lane's item of a batch, and its row there
        const uint32_t served = max(1, (p.groups - warp + PRODUCERS - 1) / PRODUCERS), depth = p.stages / p.groups;
        auto item_of = [&](uint32_t turn, uint32_t &group, uint32_t &round) {
            round = turn / served;
            group = warp + PRODUCERS * (turn - round * served);
            return blockIdx.x + gridDim.x * (round * p.groups + group);
        };
        auto fetch = [&](uint32_t first, int &pos, float &w) {
            uint32_t group, round;
            const uint32_t item = item_of(first + of, group, round);
            const int64_t t = (int64_t)(item / segments) * p.tokens + row / k;
            pos = -1;
            w = 1.f;
            if (of < batch && item < items && t < a.tokens) {
                pos = ptx::ld_dependent(a.positions + t * a.positions_ld + row % k);
                if (a.weights) w = ptx::ld_dependent(a.weights + t * a.weights_ld + row % k);
            }
        };
        int pos, next_pos, last_pos;
        float w, next_w, last_w;
        fetch(0, pos, w);
        fetch(batch, next_pos, next_w);
        bool more = warp < p.groups;
        for (uint32_t first = 0; more; first += batch) {
            fetch(first + 2 * batch, last_pos, last_w);
            const bool there = (uint32_t)pos < kept;
            const uint32_t all = __ballot_sync(0xffffffffu, there);
            for (int b = 0; b < batch; ++b) {
                uint32_t group, round;
                const uint32_t item = item_of(first + b, group, round), part = item / segments;
                if (item >= items) {
                    more = false;
                    break;
                }
                const uint32_t turns = round / depth, stage = group + p.groups * (round - turns * depth);
                const int64_t t0 = (int64_t)part * p.tokens, col = (int64_t)(item - part * segments) * segment;
                const uint32_t cols = (uint32_t)min((int64_t)segment, a.cols - col);
                const int tokens = (int)min((int64_t)p.tokens, a.tokens - t0);
                const uint32_t mask = (all >> (b * rows)) & (rows == 32 ? 0xffffffffu : (1u << rows) - 1);
                if (!__all_sync(0xffffffffu, ptx::mbar_wait(&empty[stage], ~turns & 1))) {
                    failed = true;
                    more = false;
                    break;
                }
                if (of == b) weights[stage][row] = DROP ? w * a.drop.scale : w; // (one product a row instead of one an element)
                if (lane == 0) present[stage] = mask;
                __syncwarp();
                if (lane == 0)
                    ptx::mbar_arrive_expect_tx(&full[stage], __popc(mask) * cols * (uint32_t)sizeof(S) + (a.residual ? tokens * cols * (uint32_t)sizeof(D) : 0));
                __syncwarp();
                char *at = ring + stage * p.stage_bytes;
                if (of == b && there)
                    ptx::bulk_load(at + row * p.stride * (int)sizeof(S), (const S *)a.src + (int64_t)pos * a.cols + col, cols * (uint32_t)sizeof(S), &full[stage]);
                if (a.residual && lane < tokens)
                    ptx::bulk_load(at + p.residuals + lane * p.stride * (int)sizeof(D), (const D *)a.residual + (t0 + lane) * a.residual_ld + col,
                            cols * (uint32_t)sizeof(D), &full[stage]);
            }
            pos = next_pos;
            w = next_w;
            next_pos = last_pos;
            next_w = last_w;
        }
    } else {
        uint64_t seed = 0, offset = 0;
        if constexpr (DROP) {
            seed = ld_dependent_u64(a.drop.seed);
            offset = ld_dependent_u64(a.drop.seed + 1);
        }
        const int group = (warp - PRODUCERS) / BULK_WARPS, part = (warp - PRODUCERS) % BULK_WARPS;
        const int token = part / p.warps; // the warp's token of an item
        const int mine = (part - token * p.warps) * WARP_COLS + lane * 8; // and its first column of the segment; more 256 on
        // A wait knows a phase by its parity only, so nobody may come to a stage's next phase before its last has ended: the
        // stages of a group are its own, and it has seen them end.
        int stage = group;
        uint32_t phase = 0;
        for (uint32_t item = group < p.groups ? blockIdx.x + gridDim.x * group : items; item < items; item += gridDim.x * p.groups) {
            const uint32_t q = item / segments;
            const int64_t t = (int64_t)q * p.tokens + token, col = (int64_t)(item - q * segments) * segment + mine;
            const bool work = token < p.tokens && t < a.tokens;
            const bool on[2] = {work && col < a.cols, work && col + 256 < a.cols};
            float acc[2][8];
#pragma unroll
            for (int n = 0; n < 16; ++n) acc[n / 8][n % 8] = 0.f;
            Cols<D, true> res[2];
            if (!__all_sync(0xffffffffu, ptx::mbar_wait(&full[stage], phase))) {
                failed = true;
                break;
            }
            if (work) {
                const char *at = ring + stage * p.stage_bytes;
                const S *rows = (const S *)at + token * a.choices * p.stride + mine;
                const float *w = &weights[stage][token * a.choices];
                const uint32_t there = present[stage] >> (token * a.choices);
                auto add = [&](int j) {
                    const float wj = w[j];
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        if (on[h]) {
                            Cols<S, true> x;
                            x.load_shared(rows + j * p.stride + 256 * h);
                            float v[8];
                            x.get(v);
#pragma unroll
                            for (int n = 0; n < 8; n += 2) fma2(acc[h][n], acc[h][n + 1], wj, v[n], v[n + 1]);
                        }
                };
                const uint32_t every = (1u << a.choices) - 1;
                if ((there & every) == every) {
                    int j = 0;
                    for (; j + 4 <= a.choices; j += 4) {
                        add(j);
                        add(j + 1);
                        add(j + 2);
                        add(j + 3);
                    }
                    for (; j < a.choices; ++j) add(j);
                } else {
                    for (int j = 0; j < a.choices; ++j)
                        if ((there >> j) & 1) add(j);
                }
                if (a.residual)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        if (on[h]) res[h].load_shared((const D *)(at + p.residuals) + token * p.stride + mine + 256 * h);
            }
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(&empty[stage]);
            if constexpr (DROP) {
                if (on[0]) {
                    uint32_t u[2][8];
                    random_words<true>(u[0], seed, offset, t, a.cols, col, nullptr);
                    random_words<true>(u[1], seed, offset, t, a.cols, col + 256, nullptr);
                    drop(acc[0], u[0], a.drop);
                    drop(acc[1], u[1], a.drop);
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)
                if (on[h]) {
                    if (a.residual) {
                        float v[8];
                        res[h].get(v);
#pragma unroll
                        for (int n = 0; n < 8; ++n) acc[h][n] += v[n];
                    }
                    Cols<D, true>::store((D *)a.dst + t * a.dst_ld, col + 256 * h, a.cols, acc[h]);
                }
            stage += p.groups;
            if (stage >= p.stages) {
                stage = group;
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
    const int64_t kept = rows_of_groups(a);
    const int64_t end = a.rows * a.cols;
    S *p = (S *)a.diff_src;
    constexpr int STEP = VEC ? 16 / sizeof(S) : 1;
    for (int64_t i = kept * a.cols + ((int64_t)blockIdx.x * 256 + threadIdx.x) * STEP; i < end; i += (int64_t)gridDim.x * 256 * STEP) {
        if constexpr (VEC) *reinterpret_cast<uint4 *>(p + i) = make_uint4(0, 0, 0, 0);
        else p[i] = from_f32<S>(0.f);
    }
}

// Rows of the groups that no slot names - a program took their positions back after dispatch - have a gradient of zero.  The
// first CTAs of the grid look for them while the others work on tokens: each goes through all positions and marks those of its
// part of the rows in shared memory.  Marked rows are the tokens', unmarked ones its own, so nothing is written twice.
// What a CTA takes grows with all positions, whatever its part: 32 CTAs, more only where the marks would not fit.  (us a call,
// without / with: 4096 x 8 rows of 4096 bf16 89.0 / 88.4, of 512 12.6 / 12.3, of 128 7.9 / 9.1; 131072 x 8 of 128 214 / 223.)
constexpr int MARK_ROWS = 32768; // of a CTA at most
inline unsigned mark_ctas(int64_t rows) {
    return (unsigned)std::max((rows + MARK_ROWS - 1) / MARK_ROWS, std::min<int64_t>(32, (rows + 255) / 256));
}

template <typename S, bool VEC> __device__ __forceinline__ void zero_unnamed(const CombineArgs &a, uint32_t *marks) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    const uint32_t part = ((uint32_t)((a.rows + a.mark_ctas - 1) / a.mark_ctas) + 31) / 32 * 32, first = blockIdx.x * part;
    const uint32_t kept = rows_of_groups(a); // (not waited for before the positions)
    for (uint32_t i = threadIdx.x; i < part / 32; i += 256) marks[i] = 0;
    __syncthreads();
    auto mark = [&](uint32_t position) {
        const uint32_t at = position - first;
        if (at < part) atomicOr(&marks[at / 32], 1u << (at % 32));
    };
    const uint32_t slots = (uint32_t)(a.tokens * a.choices);
    uint32_t done = 0;
    if (a.positions_ld == a.choices && (uintptr_t)a.positions % 16 == 0) {
        constexpr int FLIGHT = 8; // of four each
        for (uint32_t q = threadIdx.x; q < slots / 4; q += 256 * FLIGHT) {
            uint4 at[FLIGHT];
#pragma unroll
            for (int f = 0; f < FLIGHT; ++f) {
                at[f] = make_uint4(~0u, ~0u, ~0u, ~0u);
                if (q + 256 * f < slots / 4) at[f] = ptx::ld_dependent((const uint4 *)a.positions + q + 256 * f);
            }
#pragma unroll
            for (int f = 0; f < FLIGHT; ++f) {
                mark(at[f].x);
                mark(at[f].y);
                mark(at[f].z);
                mark(at[f].w);
            }
        }
        done = slots / 4 * 4;
    }
    constexpr int FLIGHT = 16;
    for (uint32_t s0 = done + threadIdx.x; s0 < slots; s0 += 256 * FLIGHT) {
        uint32_t at[FLIGHT];
#pragma unroll
        for (int f = 0; f < FLIGHT; ++f) {
            const uint32_t s = s0 + 256 * f, t = s / (uint32_t)a.choices;
            at[f] = ~0u;
            if (s < slots) at[f] = (uint32_t)ptx::ld_dependent(a.positions + (int64_t)t * a.positions_ld + (s - t * (uint32_t)a.choices));
        }
#pragma unroll
        for (int f = 0; f < FLIGHT; ++f) mark(at[f]);
    }
    __syncthreads();
    const uint32_t count = kept > first ? min(part, kept - first) : 0;
    for (uint32_t w = warp; w * 32 < count; w += 8) {
        uint32_t gone = ~marks[w] & (count - w * 32 >= 32 ? 0xffffffffu : (1u << (count - w * 32)) - 1);
        for (; gone; gone &= gone - 1) {
            S *row = (S *)a.diff_src + (int64_t)(first + w * 32 + __ffs(gone) - 1) * a.cols;
            constexpr int STEP = VEC ? 16 / sizeof(S) : 1;
            for (int64_t c = lane * STEP; c < a.cols; c += 32 * STEP) {
                if constexpr (VEC) *reinterpret_cast<uint4 *>(row + c) = make_uint4(0, 0, 0, 0);
                else row[c] = from_f32<S>(0.f);
            }
        }
    }
}

// CTAs per SM that the gradient's registers are cut to (0: the compiler's choice).  us a call, 4096 tokens, the same inputs every
// call, uncut / cut: bf16 with dropout, eight rows of 4096 106.4 / 88.5 (three; 97.9 four), four rows of 4096 51.5 / 47.7 (five);
// rows that start anywhere, bf16, two of 2047 without dropout 21.9 / 20.7 (five); f32, eight rows of 512 with dropout 27.0 / 25.4
// (two), of 255 without 12.9 / 11.4.  Elsewhere a cut gains nothing or costs: rows that start anywhere, bf16 with dropout, eight of
// 2047 81.2 / 82.4 (three), 101.6 (two), four of 2047 48.7 / 71.3 (two); f32, two of 4096 with dropout 53.0 / 67.5 (two).
template <typename S, typename D, bool VEC, bool DROP, int GROUP, int THREADS>
constexpr int GRADIENT_CTAS = !VEC && !DROP && GROUP == 2 ? 5
        : sizeof(S) == 4 && GROUP == 8 && THREADS == 32   ? 2
        : !VEC || sizeof(S) == 4 || THREADS == 32         ? 0
        : GROUP == 8                                      ? 3
        : GROUP == 4 && sizeof(D) == 2                    ? 5
                                                          : 0;

// THREADS of the 256 of a CTA work on a token: all of them, or a warp where rows are short.
template <typename S, typename D, bool VEC, bool DROP, int THREADS, int GROUP>
__global__ void __launch_bounds__(256, GRADIENT_CTAS<S, D, VEC, DROP, GROUP, THREADS>) combine_backward_kernel(const __grid_constant__ CombineArgs a) {
    __shared__ __align__(16) uint32_t words[DROP && !VEC ? 8 * 128 : 4];
    __shared__ float partial[8][GROUP];
    __shared__ uint32_t marks[MARK_ROWS / 32];
    ptx::grid_dependency_wait();
    constexpr int N = Cols<S, VEC>::N;
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    const uint32_t block = blockIdx.x - a.mark_ctas; // (wraps beyond all tokens for the CTAs that mark)
    const int64_t t = THREADS == 256 ? (int64_t)block : (int64_t)block * 8 + warp;
    const int64_t units = (row_units<VEC>(a.cols, DROP) + 31) / 32 * 32;
    if (t < a.tokens) {
        uint64_t seed = 0, offset = 0;
        if constexpr (DROP) {
            seed = ld_dependent_u64(a.drop.seed);
            offset = ld_dependent_u64(a.drop.seed + 1);
        }
        const uint32_t kept = rows_of_groups(a);
        // lane j: position and weight of choice j
        const int my_pos = lane < a.choices ? ptx::ld_dependent(a.positions + t * a.positions_ld + lane) : -1;
        const float my_w = lane < a.choices ? ptx::ld_dependent(a.weights + t * a.weights_ld + lane) : 0.f;
        for (int j0 = 0; j0 < a.choices; j0 += GROUP) {
            float dot[GROUP];
#pragma unroll
            for (int j = 0; j < GROUP; ++j) dot[j] = 0.f;
            for (int64_t u = threadIdx.x % THREADS; u < units; u += THREADS) {
                const int64_t col = unit_column<VEC>(u, t, a.cols, DROP);
                Cols<D, VEC> g;
                Cols<S, VEC> x[GROUP];
                g.load((const D *)a.diff_dst + t * a.diff_dst_ld, col, a.cols);
#pragma unroll
                for (int j = 0; j < GROUP; ++j) {
                    const uint32_t pos = __shfl_sync(0xffffffffu, my_pos, j0 + j);
                    if (pos < kept) x[j].load((const S *)a.src + (int64_t)pos * a.cols, col, a.cols);
                }
                float dy[N];
                g.get(dy);
                if constexpr (DROP) apply_dropout<VEC>(dy, a.drop, seed, offset, t, a.cols, col, words + (VEC ? 0 : warp * 128));
#pragma unroll
                for (int j = 0; j < GROUP; ++j) {
                    const uint32_t pos = __shfl_sync(0xffffffffu, my_pos, j0 + j);
                    const float w = __shfl_sync(0xffffffffu, my_w, j0 + j);
                    if (pos < kept) {
                        float v[N], d[N];
                        x[j].get(v);
#pragma unroll
                        for (int n = 0; n < N; ++n) {
                            dot[j] = fmaf(dy[n], v[n], dot[j]);
                            d[n] = w * dy[n];
                        }
                        Cols<S, VEC>::store((S *)a.diff_src + (int64_t)pos * a.cols, col, a.cols, d);
                    }
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
    if (blockIdx.x < a.mark_ctas) zero_unnamed<S, VEC>(a, marks);
    zero_tail<S, VEC>(a);
}

template <typename S, typename D, bool DROP> int launch_bulk(const CombineArgs &a, int sm_count, cudaStream_t st) {
    BulkPlan p {};
    p.a = a;
    const int row = a.choices * (int)sizeof(S) + (a.residual ? (int)sizeof(D) : 0); // bytes per column of a token
    const int most = BULK_RING / 4; // four stages at least
    p.warps = (int)std::min<int64_t>(BULK_WARPS, (a.cols + WARP_COLS - 1) / WARP_COLS);
    while (p.warps > 1 && row * p.warps * WARP_COLS > most) --p.warps;
    p.segments = (uint32_t)((a.cols + p.warps * WARP_COLS - 1) / (p.warps * WARP_COLS));
    p.stride = p.segments == 1 ? (int)((a.cols + 7) / 8 * 8) : p.warps * WARP_COLS;
    p.tokens = p.segments == 1 ? std::min(BULK_WARPS / p.warps, 32 / a.choices) : 1;
    while (p.tokens > 1 && row * p.tokens * p.stride > most) --p.tokens;
    p.residuals = p.tokens * a.choices * p.stride * (int)sizeof(S);
    p.stage_bytes = p.tokens * row * p.stride;
    const int room = std::min(BULK_MAX_STAGES, BULK_RING / p.stage_bytes);
    p.groups = std::min(room, BULK_GROUPS);
    for (int g = p.groups - 1; g >= 4 && g > p.groups - 6; --g) // as many as leave the least of the ring unused
        if (room / g * g > room / p.groups * p.groups) p.groups = g;
    p.stages = room / p.groups * p.groups;
    p.items = (uint32_t)((a.tokens + p.tokens - 1) / p.tokens * p.segments);
    static std::atomic<unsigned long long> done;
    if (!opt_in_dynamic_smem(combine_bulk_kernel<S, D, DROP>, BULK_RING, done)) return 5;
    return launch_dependent(combine_bulk_kernel<S, D, DROP>, p, std::min<unsigned>(p.items, sm_count), BULK_THREADS, BULK_RING, st);
}

template <typename S, typename D, bool DROP> int launch_forward(const CombineArgs &a, bool vec, int sm_count, cudaStream_t st) {
    const int64_t total = a.tokens * (vec ? row_units<true>(a.cols, DROP) : row_units<false>(a.cols, DROP));
    const int64_t grid = (total + 255) / 256;
    // The ring's start and the number of its copies cost more than they give where a row is below 2 KB, where there are few
    // sums, most of all with one or two rows a token, and, with many rows, where a stage leaves the ring few others.
    // us a call, residual, no dropout, thread by thread / ring (up to eight rows: inputs that are not in L2)
    //   rows     bf16                                                       f32
    //    1       4096 x 1024 7.9 / 8.2, 8192 x 1024 13.0 / 12.1,            8192 x 1024 19.4 / 19.7, 8192 x 4096 69.6 / 68.0
    //            4096 x 4096 23.2 / 18.8
    //    2       8192 x 1024 14.5 / 15.7, 8192 x 4096 49.2 / 49.2           8192 x 2048 42.0 / 45.0
    //            (with dropout 73.1 / 71.2), 6997 x 7936 without residual
    //            88.1 / 84.5
    //    4       1024 x 1024 6.3 / 6.0, 8192 x 4096 99.3 / 68.0             1024 x 1024 7.3 / 8.8, 4096 x 512 12.4 / 11.8,
    //                                                                       8192 x 4096 147 / 125
    //    8       1024 x 1024 7.6 / 7.8, 512 x 4096 11.5 / 11.1,             2048 x 512 10.0 / 10.8, 8192 x 2048 101.5 / 103.1
    //            8192 x 4096 124.5 / 101.9, 4096 x 512 7.4 / 9.0            (with dropout 106.6 / 106.5)
    //   12       2730 x 4096 61.8 / 52.8                                    2730 x 4096 97.9 / 97.8
    //   16       4096 x 2048 54.2 / 61.4, 2048 x 4096 54.0 / 52.7           2048 x 4096 90.3 / 93.4
    //   32       1024 x 4096 49.8 / 68.0                                    1024 x 4096 84.7 / 100.7
    const int64_t sums = a.tokens * a.cols;
    const bool many = a.choices == 1 ? sums >= 1 << 23 : a.choices == 2 ? sizeof(S) == 2 && sums >= 1 << 25 : a.choices <= 12 && sums >= 1 << 21;
    if (vec && a.cols * (int64_t)sizeof(S) >= 2048 && many
            && a.tokens * ((a.cols + WARP_COLS - 1) / WARP_COLS) < (1 << 30) && !a.drop.drop_all)
        return launch_bulk<S, D, DROP>(a, sm_count, st);
    if (grid > 0x7fffffff) return 3;
    // (3000 x 2 x 2047 bf16 with groups of eight rows 23.5 us / of two 14.4; four rows in groups of eight / of four: 400 x 4096 bf16
    // with dropout 6.8 / 6.2, 3000 x 2047 bf16 25.5 / 25.8, f32 33.1 / 30.0: not worth their kernels)
    void (*kernel)(CombineArgs) = a.choices <= 2 ? (vec ? combine_kernel<S, D, true, DROP, 2> : combine_kernel<S, D, false, DROP, 2>)
                                                 : (vec ? combine_kernel<S, D, true, DROP, 8> : combine_kernel<S, D, false, DROP, 8>);
    return launch_dependent(kernel, a, (unsigned)grid, 256, 0, st);
}

template <typename S, typename D, bool VEC, bool DROP, int GROUP> int launch_backward(const CombineArgs &a, cudaStream_t st) {
    const bool wide = row_units<VEC>(a.cols, DROP) > 64;
    CombineArgs b = a;
    b.mark_ctas = mark_ctas(a.rows);
    const int64_t grid = (wide ? a.tokens : (a.tokens + 7) / 8) + b.mark_ctas;
    if (grid > 0x7fffffff) return 3;
    return launch_dependent(wide ? combine_backward_kernel<S, D, VEC, DROP, 256, GROUP> : combine_backward_kernel<S, D, VEC, DROP, 32, GROUP>, b,
            (unsigned)grid, 256, 0, st);
}
template <typename S, typename D, bool DROP> int launch_backward(const CombineArgs &a, bool vec, cudaStream_t st) {
    if (a.choices <= 2) return vec ? launch_backward<S, D, true, DROP, 2>(a, st) : launch_backward<S, D, false, DROP, 2>(a, st);
    if (a.choices <= 4) return vec ? launch_backward<S, D, true, DROP, 4>(a, st) : launch_backward<S, D, false, DROP, 4>(a, st);
    return vec ? launch_backward<S, D, true, DROP, 8>(a, st) : launch_backward<S, D, false, DROP, 8>(a, st);
}

template <typename S, typename D> int launch_types(const CombineArgs &a, bool backward, int sm_count, cudaStream_t st) {
    const bool drop = a.drop.seed != nullptr;
    const int64_t ds = sizeof(D);
    bool vec = a.cols % 8 == 0 && rows_aligned(a.src, a.cols * (int64_t)sizeof(S), a.rows);
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

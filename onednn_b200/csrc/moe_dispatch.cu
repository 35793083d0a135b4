// Tokens into grouped memory: a stable sort of the n = tokens x choices slots by expert (slot = token * choices + choice),
// and the tokens' rows copied to their slots' places.
//   offsets[e] = number of slots whose expert is <= e, position[slot] = offsets[e - 1] + slots of e before this one
// A slot whose index names no expert has position -1 and no row; the rows behind the last group are zeros.
//
// A counting sort with one digit, the expert.  A CTA takes a contiguous range of tokens: it needs the counts of all slots
// (where each group begins) and of the slots before its range; inside, 32 slots at a time are ranked by matching lanes.
// A token's row is read once and stored to its places, so the copy moves (1 + choices) rows per token and its writes
// bound it.  Few slots: every CTA counts and ranks all of them itself, one launch.  More: a first kernel leaves the counts
// of every range, a second adds them up.
#include <algorithm>

#include "launch.h"
#include "token_rows.cuh"

namespace qmm {

namespace {

constexpr int THREADS = 1024, WARPS = THREADS / 32;
constexpr int TILE = 1024; // slots ranked at a time
constexpr int SHARED_BYTES = 220 * 1024; // dynamic, at most
constexpr int DIRECT_SLOTS = 2048; // up to here every CTA ranks all slots

// Rows that bulk copies can move: some warps of a CTA each stream segments of rows through a ring of their own in shared
// memory, one load in and a store to every place out, so that no register or instruction stands between.
constexpr int MOVERS = 8, SLOTS = 3;
constexpr int SLOT_BYTES = 8192;

struct Plan {
    DispatchArgs a;
    int *counts; // [ranges][experts], of the ranges of tokens
    int ranges, range_tokens;
    int segment, segments; // bulk copies: bytes of a segment (0: none), segments of a row
    int ring; // where their rings begin in the dynamic shared memory
};

// One mover's ring; the whole warp calls it.
struct Mover {
    const Plan &p;
    char *ring;
    uint64_t *full; // [SLOTS]
    int lane, mover;
    int slot = 0; // next to be used
    uint32_t phases = 0; // parity of each slot
    bool failed = false;

    __device__ __forceinline__ void load(int64_t item, int64_t t0, int at) {
        if (lane != 0) return;
        const int64_t t = t0 + item / p.segments;
        const int from = (int)(item % p.segments) * p.segment, bytes = (int)min((int64_t)p.segment, p.a.row_bytes - from);
        ptx::mbar_arrive_expect_tx(&full[at], bytes);
        ptx::bulk_load(ring + at * p.segment, p.a.src + t * p.a.src_pitch + from, bytes, &full[at]);
    }
    // the loads of a tile's first items
    __device__ __forceinline__ void begin(int64_t t0, int64_t items) {
#pragma unroll
        for (int q = 0; q < SLOTS - 1; ++q)
            if (mover + q * MOVERS < items && !failed) load(mover + q * MOVERS, t0, (slot + q) % SLOTS);
    }
    __device__ __forceinline__ void move(int64_t t0, int64_t items, const int *place) {
        for (int64_t i = mover; i < items && !failed; i += MOVERS) {
            if (!__all_sync(0xffffffffu, ptx::mbar_wait(&full[slot], (phases >> slot) & 1))) {
                failed = true;
                break;
            }
            phases ^= 1u << slot;
            const int t = (int)(i / p.segments), from = (int)(i % p.segments) * p.segment;
            const int to = lane < p.a.choices ? place[t * p.a.choices + lane] : -1;
            if (to >= 0)
                ptx::bulk_store(p.a.dst + (int64_t)to * p.a.row_bytes + from, ring + slot * p.segment, (uint32_t)min((int64_t)p.segment, p.a.row_bytes - from));
            ptx::bulk_commit();
            // the slot of the item before is free once its stores have read it
            ptx::bulk_wait_read<1>();
            __syncwarp();
            const int64_t ahead = i + (SLOTS - 1) * MOVERS;
            if (ahead < items) load(ahead, t0, (slot + SLOTS - 1) % SLOTS);
            slot = (slot + 1) % SLOTS;
        }
    }
};

__device__ __forceinline__ int slot_expert(const DispatchArgs &a, int slot) {
    const int t = slot / a.choices;
    const int e = ptx::ld_dependent(a.indices + (int64_t)t * a.indices_ld + (slot - t * a.choices));
    return (unsigned)e < (unsigned)a.experts ? e : -1;
}

__global__ void __launch_bounds__(THREADS) dispatch_count_kernel(const __grid_constant__ Plan p) {
    __shared__ int count[TOKEN_MAX_EXPERTS];
    ptx::grid_dependency_wait();
    const DispatchArgs &a = p.a;
    for (int e = threadIdx.x; e < a.experts; e += THREADS) count[e] = 0;
    __syncthreads();
    const int64_t begin = (int64_t)blockIdx.x * p.range_tokens;
    const int64_t end = begin + p.range_tokens < a.tokens ? begin + p.range_tokens : a.tokens;
    for (int64_t s = begin * a.choices + threadIdx.x; s < end * a.choices; s += THREADS) {
        const int e = slot_expert(a, (int)s);
        if (e >= 0) atomicAdd(&count[e], 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < a.experts; e += THREADS) p.counts[(int64_t)blockIdx.x * a.experts + e] = count[e];
}

// Copies unit `u` (of U's size) of a token's row to the places in `place`.
template <typename U> __device__ __forceinline__ void store_unit(const DispatchArgs &a, U v, int64_t u, const int *place) {
    for (int j = 0; j < a.choices; ++j)
        if (place[j] >= 0) *((U *)(a.dst + (int64_t)place[j] * a.row_bytes) + u) = v;
}

template <typename U, bool DIRECT, bool BULK> __global__ void __launch_bounds__(THREADS) dispatch_kernel(const __grid_constant__ Plan p) {
    extern __shared__ __align__(128) int shared[];
    __shared__ int scan[WARPS], kept;
    __shared__ uint64_t full[MOVERS][SLOTS];
    const DispatchArgs &a = p.a;
    int *base = shared, *total = base + a.experts; // per expert: next free place, number of slots
    int *place = total + a.experts; // positions of a tile's slots (DIRECT: of all slots)
    unsigned short *table = (unsigned short *)(place + (DIRECT ? DIRECT_SLOTS : TILE)); // [warp][expert]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid / 32;
    const int n = a.tokens * a.choices;
    // the tokens whose positions this CTA writes down, and (not DIRECT) whose rows it moves
    const int first = DIRECT ? (int)((int64_t)a.tokens * blockIdx.x / gridDim.x) : blockIdx.x * p.range_tokens;
    const int last = DIRECT ? (int)((int64_t)a.tokens * (blockIdx.x + 1) / gridDim.x)
                            : (int)min((int64_t)a.tokens, (int64_t)first + p.range_tokens);
    const int tile_tokens = TILE / a.choices;
    if (BULK && tid == 0) {
        for (int i = 0; i < MOVERS * SLOTS; ++i) ptx::mbar_init(&full[0][0] + i, 1);
        ptx::fence_barrier_init();
    }
    __syncthreads();
    ptx::grid_dependency_wait();
    Mover mover {p, (char *)shared + p.ring + warp * (SLOTS * p.segment), full[BULK ? warp % MOVERS : 0], lane, warp};
    if (BULK && warp < MOVERS) mover.begin(first, (int64_t)min(tile_tokens, last - first) * p.segments);

    for (int e = tid; e < a.experts; e += THREADS) base[e] = total[e] = 0;
    __syncthreads();
    if constexpr (DIRECT) {
        for (int s = tid; s < n; s += THREADS) {
            const int e = slot_expert(a, s);
            if (e >= 0) atomicAdd(&total[e], 1);
        }
    } else {
        // threads beside one another take neighbouring experts, groups of them every few ranges
        const int width = (a.experts + 31) / 32 * 32, step = THREADS / width, e = tid % width;
        if (e < a.experts && tid < step * width) {
            int before = 0, all = 0;
            for (int r = tid / width; r < p.ranges; r += step) {
                const int c = ptx::ld_dependent(p.counts + (int64_t)r * a.experts + e);
                all += c;
                before += r < (int)blockIdx.x ? c : 0;
            }
            atomicAdd(&total[e], all);
            atomicAdd(&base[e], before);
        }
    }
    __syncthreads();
    { // where each group begins: sums over the experts before it (one thread per expert)
        const int mine = tid < a.experts ? total[tid] : 0;
        int sum = mine;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const int v = __shfl_up_sync(0xffffffffu, sum, d);
            if (lane >= d) sum += v;
        }
        if (lane == 31) scan[warp] = sum;
        __syncthreads();
        if (warp == 0) {
            int v = scan[lane];
#pragma unroll
            for (int d = 1; d < 32; d *= 2) {
                const int x = __shfl_up_sync(0xffffffffu, v, d);
                if (lane >= d) v += x;
            }
            scan[lane] = v;
        }
        __syncthreads();
        if (warp > 0) sum += scan[warp - 1];
        if (tid < a.experts) {
            base[tid] += sum - mine;
            if (blockIdx.x == 0) a.offsets[tid] = sum;
            if (tid == a.experts - 1) kept = sum;
        }
    }
    __syncthreads();

    const int64_t units = a.row_bytes / sizeof(U);
    for (int t0 = DIRECT ? 0 : first; t0 < (DIRECT ? a.tokens : last); t0 += tile_tokens) {
        const int t1 = min(t0 + tile_tokens, DIRECT ? a.tokens : last), slots = (t1 - t0) * a.choices;
        const int warps = (slots + 31) / 32;
        for (int i = tid; i < warps * a.experts; i += THREADS) table[i] = 0;
        const int slot = t0 * a.choices + tid;
        const int e = tid < slots ? slot_expert(a, slot) : -1;
        __syncthreads();
        const unsigned same = __match_any_sync(0xffffffffu, e);
        const int rank = __popc(same & ((1u << lane) - 1));
        if (e >= 0 && rank == 0) table[warp * a.experts + e] = (unsigned short)__popc(same);
        __syncthreads();
        int tile_count = 0;
        if (tid < a.experts)
            for (int w = 0; w < warps; ++w) {
                const int c = table[w * a.experts + tid];
                table[w * a.experts + tid] = (unsigned short)tile_count;
                tile_count += c;
            }
        __syncthreads();
        if (tid < slots) {
            const int pos = e >= 0 ? base[e] + table[warp * a.experts + e] + rank : -1;
            place[(DIRECT ? t0 * a.choices : 0) + tid] = pos;
            const int t = slot / a.choices;
            if (t >= first && t < last) a.positions[(int64_t)t * a.positions_ld + (slot - t * a.choices)] = pos;
        }
        __syncthreads();
        if (tid < a.experts) base[tid] += tile_count;
        if constexpr (BULK) {
            if (warp < MOVERS) {
                const int64_t items = (int64_t)(t1 - t0) * p.segments;
                if (t0 != first) mover.begin(t0, items);
                mover.move(t0, items, place);
            }
        } else if constexpr (!DIRECT) {
            const int64_t work = (int64_t)(t1 - t0) * units;
            constexpr int FLIGHT = 4;
            for (int64_t i0 = tid; i0 < work; i0 += (int64_t)THREADS * FLIGHT) {
                U v[FLIGHT];
                int64_t t[FLIGHT], u[FLIGHT];
#pragma unroll
                for (int f = 0; f < FLIGHT; ++f) {
                    const int64_t i = i0 + f * THREADS;
                    t[f] = work <= 0xffffffff ? (uint32_t)i / (uint32_t)units : i / units;
                    u[f] = i - t[f] * units;
                    if (i < work) v[f] = *((const U *)(a.src + (t0 + t[f]) * a.src_pitch) + u[f]);
                }
#pragma unroll
                for (int f = 0; f < FLIGHT; ++f)
                    if (i0 + f * THREADS < work) store_unit(a, v[f], u[f], place + t[f] * a.choices);
            }
        }
        __syncthreads();
    }
    if constexpr (DIRECT) {
        const int64_t work = a.tokens * units;
        for (int64_t i = (int64_t)blockIdx.x * THREADS + tid; i < work; i += (int64_t)gridDim.x * THREADS) {
            const int64_t t = i / units, u = i - t * units;
            store_unit(a, *((const U *)(a.src + t * a.src_pitch) + u), u, place + t * a.choices);
        }
    }
    U zero;
    memset(&zero, 0, sizeof(U));
    const int64_t tail = (int64_t)(n - kept) * units;
    U *behind = (U *)(a.dst + (int64_t)kept * a.row_bytes);
    for (int64_t i = (int64_t)blockIdx.x * THREADS + tid; i < tail; i += (int64_t)gridDim.x * THREADS) behind[i] = zero;
    if (BULK && warp < MOVERS) {
        ptx::bulk_wait_all();
        if (mover.failed) { // a load may still be on its way: it lands before the memory goes
            for (int s = 0; s < SLOTS; ++s)
                for (int parity = 0; parity < 2; ++parity) (void)ptx::mbar_wait(&mover.full[s], parity, 500000000ull);
            if (lane == 0 && a.status) atomicExch(a.status, 5);
        }
    }
}

size_t plan_bytes(int experts, bool direct) {
    return experts * (2 * sizeof(int) + WARPS * sizeof(short)) + (direct ? DIRECT_SLOTS : TILE) * sizeof(int);
}

template <typename U, bool DIRECT, bool BULK> int launch_kernel(const Plan &p, size_t smem, unsigned grid, cudaStream_t st) {
    static std::atomic<unsigned long long> done;
    if (!opt_in_dynamic_smem(dispatch_kernel<U, DIRECT, BULK>, SHARED_BYTES, done)) return 5;
    return launch_dependent(dispatch_kernel<U, DIRECT, BULK>, p, grid, THREADS, smem, st);
}

template <typename U> int launch_unit(Plan &p, bool direct, unsigned grid, cudaStream_t st) {
    const size_t plan = plan_bytes(p.a.experts, direct);
    if (direct) return launch_kernel<U, true, false>(p, plan, grid, st);
    if constexpr (sizeof(U) == 16) {
        if (p.a.row_bytes >= 512) {
            p.ring = (int)((plan + 127) / 128 * 128);
            const int64_t most = std::min<int64_t>(SLOT_BYTES, (SHARED_BYTES - p.ring) / (MOVERS * SLOTS) / 128 * 128);
            // rows in equal segments, and segments enough for every mover of a short range
            const int64_t wanted = std::max<int64_t>((p.a.row_bytes + most - 1) / most,
                    std::min<int64_t>((MOVERS + p.range_tokens - 1) / p.range_tokens, p.a.row_bytes / 1024));
            p.segment = (int)(((p.a.row_bytes + wanted - 1) / wanted + 127) / 128 * 128);
            p.segments = (int)((p.a.row_bytes + p.segment - 1) / p.segment);
            return launch_kernel<U, false, true>(p, p.ring + MOVERS * SLOTS * p.segment, grid, st);
        }
    }
    return launch_kernel<U, false, false>(p, plan, grid, st);
}

} // namespace

// counts of up to `sm_count` ranges
size_t dispatch_scratch_bytes(int experts, int sm_count) { return (size_t)experts * sm_count * sizeof(int); }

int launch_dispatch(const DispatchArgs &a, int *scratch, int sm_count, cudaStream_t st) {
    Plan p {};
    p.a = a;
    if (a.tokens == 0) // no slots: the groups are empty, and say so
        return cudaMemsetAsync(a.offsets, 0, a.experts * sizeof(int), st) == cudaSuccess ? 0 : 5;
    // the widest unit that every row starts and ends on
    const uint64_t places = (uint64_t)a.row_bytes | (uint64_t)(uintptr_t)a.dst | (uint64_t)(uintptr_t)a.src
            | (a.tokens > 1 ? (uint64_t)a.src_pitch : 0);
    const int unit = places % 16 == 0 ? 16 : places % 4 == 0 ? 4 : places % 2 == 0 ? 2 : 1;
    const bool direct = (int64_t)a.tokens * a.choices <= DIRECT_SLOTS;
    unsigned grid;
    if (direct) {
        const int64_t work = a.tokens * (a.row_bytes / unit);
        grid = (unsigned)std::min<int64_t>(sm_count, std::max<int64_t>(1, (work + 127) / 128));
    } else {
        p.range_tokens = (a.tokens + sm_count - 1) / sm_count;
        p.ranges = (a.tokens + p.range_tokens - 1) / p.range_tokens;
        p.counts = scratch;
        grid = p.ranges;
        const int rc = launch_dependent(dispatch_count_kernel, p, grid, THREADS, 0, st);
        if (rc) return rc;
        count_launch();
    }
    const int rc = unit == 16 ? launch_unit<uint4>(p, direct, grid, st)
            : unit == 4       ? launch_unit<uint32_t>(p, direct, grid, st)
            : unit == 2       ? launch_unit<uint16_t>(p, direct, grid, st)
                              : launch_unit<uint8_t>(p, direct, grid, st);
    if (rc == 0) count_launch();
    return rc;
}

} // namespace qmm

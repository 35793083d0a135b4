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
constexpr int DIRECT_SLOTS = 2048; // up to here every CTA ranks all slots

struct Plan {
    DispatchArgs a;
    int *counts; // [ranges][experts], of the ranges of tokens
    int ranges, range_tokens;
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

template <typename U, bool DIRECT> __global__ void __launch_bounds__(THREADS) dispatch_kernel(const __grid_constant__ Plan p) {
    extern __shared__ __align__(16) int shared[];
    __shared__ int scan[WARPS], kept;
    const DispatchArgs &a = p.a;
    int *base = shared, *total = base + a.experts; // per expert: next free place, number of slots
    int *place = total + a.experts; // positions of a tile's slots (DIRECT: of all slots)
    unsigned short *table = (unsigned short *)(place + (DIRECT ? DIRECT_SLOTS : TILE)); // [warp][expert]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid / 32;
    const int n = a.tokens * a.choices;
    ptx::grid_dependency_wait();

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
    // the tokens whose positions this CTA writes down, and (not DIRECT) whose rows it moves
    const int first = DIRECT ? (int)((int64_t)a.tokens * blockIdx.x / gridDim.x) : blockIdx.x * p.range_tokens;
    const int last = DIRECT ? (int)((int64_t)a.tokens * (blockIdx.x + 1) / gridDim.x)
                            : (int)min((int64_t)a.tokens, (int64_t)first + p.range_tokens);
    const int tile_tokens = TILE / a.choices;
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
        if constexpr (!DIRECT) {
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
}

template <typename U> int launch_unit(const Plan &p, bool direct, unsigned grid, cudaStream_t st) {
    const size_t smem = p.a.experts * (2 * sizeof(int) + WARPS * sizeof(short)) + (direct ? DIRECT_SLOTS : TILE) * sizeof(int);
    static std::atomic<unsigned long long> done_direct, done_ranges;
    const int most = TOKEN_MAX_EXPERTS * (2 * sizeof(int) + WARPS * sizeof(short)) + DIRECT_SLOTS * sizeof(int);
    auto kernel = direct ? dispatch_kernel<U, true> : dispatch_kernel<U, false>;
    if (!opt_in_dynamic_smem(kernel, most, direct ? done_direct : done_ranges)) return 5;
    return launch_dependent(kernel, p, grid, THREADS, smem, st);
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

// Tokens into grouped memory: a stable sort of the n = tokens x choices slots by expert (slot = token * choices + choice),
// and the tokens' rows copied to their slots' places.
//   offsets[e] = number of slots whose expert is <= e, position[slot] = offsets[e - 1] + slots of e before this one
// A slot whose index names no expert has position -1 and no row; the rows behind the last group are zeros.
//
// The places come from a counting sort with one digit, the expert.  A CTA takes a contiguous range of tokens: it needs the
// counts of all slots (where each group begins) and of the slots before its range, which a kernel before leaves behind;
// inside, 32 slots at a time are ranked by matching lanes.  Then a token's row is read once and stored to its places.  The
// copy moves (1 + choices) rows per token and is bound by its writes.  (Gathering in the order of the rows writes in
// sequence, but reads every token `choices` times, past L2: 16384 x 8 x 4096 bf16, places given, 295 us, this way 199.  A ring
// of bulk copies in the sorting kernel itself: 8192 x 8 x 4096 115 us in all, this way 104.)
#include <algorithm>
#include <climits>
#include <type_traits>

#include "launch.h"
#include "token_rows.cuh"

namespace qmm {

namespace {

constexpr int THREADS = 1024, WARPS = THREADS / 32;
constexpr int TILE = 1024; // slots ranked at a time
// Up to here every CTA that sorts counts all slots itself, which saves a launch (4096 slots 13.3 -> 11.4 us; 16384 32.6 -> 34.5).
constexpr int SELF_SLOTS = 8192;
// Up to here one launch does everything.  It takes about 2 us, 0.0155 for every slot (each is ranked against all) and 0.001 for
// every 100 units of the tokens' rows (a thread copies one after the other).  The other form's two launches take the device 5.6,
// where rows start anywhere 5 and 0.3 for every choice, and the host, called one by one, 6 to 7: the limit is 6.5, and 6.2 and 0.3 a
// choice.  us on the device, one launch / two, bf16: 1 x 8 x 4096 2.5 / 5.2, 37 x 2 3.2 / 6.1, 16 x 8 4.3 / 5.5, 24 x 8 5.3 / 5.6,
// 32 x 8 6.3 / 5.6 (one by one 6.5 / 6.9), 256 x 1 7.1 / 5.9; 128 x 1 x 8192 (units of 16 bytes) 5.2 / 5.8, 256 x 8192 8.3 / 6.1;
// rows that start anywhere (units of an element): 64 x 2 x 2047 5.3 / 5.6, 32 x 8 6.1 / 8.1 for 1001 and 7.6 / 7.8 for 4097,
// 128 x 2 x 1001 7.3 / 5.9, x 4097 11.2 / 5.9.
constexpr int FEW_SLOTS = 256;
inline bool few(int64_t slots, int64_t units, int choices, bool aligned) {
    return slots <= FEW_SLOTS && slots + units / 1500 <= (aligned ? 290 : 270 + 20 * choices);
}

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

// inclusive sums over the lanes
__device__ __forceinline__ int warp_scan(int v) {
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const int x = __shfl_up_sync(0xffffffffu, v, d);
        if ((int)(threadIdx.x & 31) >= d) v += x;
    }
    return v;
}

// Entries from a warp's row of the table to the next: an odd number of words, so that a column's 32 lie in different banks.
__host__ __device__ constexpr int table_pitch(int experts) { return (experts + 3) / 4 * 4 + 2; }

constexpr size_t place_bytes(int experts) { return experts * 3 * sizeof(int) + WARPS * table_pitch(experts) * sizeof(short); }

__global__ void __launch_bounds__(THREADS) dispatch_count_kernel(const __grid_constant__ Plan p) {
    __shared__ int count[TOKEN_MAX_EXPERTS];
    const DispatchArgs &a = p.a;
    for (int e = threadIdx.x; e < a.experts; e += THREADS) count[e] = 0;
    __syncthreads();
    ptx::grid_dependency_wait();
    const int64_t begin = (int64_t)blockIdx.x * p.range_tokens;
    const int64_t end = begin + p.range_tokens < a.tokens ? begin + p.range_tokens : a.tokens;
    for (int64_t s = begin * a.choices + threadIdx.x; s < end * a.choices; s += THREADS) {
        const int e = slot_expert(a, (int)s);
        if (e >= 0) atomicAdd(&count[e], 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < a.experts; e += THREADS) p.counts[(int64_t)blockIdx.x * a.experts + e] = count[e];
}

// Offsets, and the positions of a range's slots.  SELF: no counts from before.
template <bool SELF> __global__ void __launch_bounds__(THREADS) dispatch_place_kernel(const __grid_constant__ Plan p) {
    extern __shared__ __align__(16) int shared[];
    __shared__ int scan[WARPS];
    const DispatchArgs &a = p.a;
    const int pitch = table_pitch(a.experts);
    // per expert: number of slots, next free place, that of the tile at hand; per warp and expert: slots of the tile before
    int *total = shared, *base = total + a.experts, *tile_base = base + a.experts;
    unsigned short *table = (unsigned short *)(tile_base + a.experts);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid / 32;
    const int first = blockIdx.x * p.range_tokens, last = (int)min((int64_t)a.tokens, (int64_t)first + p.range_tokens);
    for (int e = tid; e < a.experts; e += THREADS) base[e] = total[e] = 0;
    __syncthreads();
    ptx::grid_dependency_wait();
    if constexpr (SELF) {
        for (int s = tid; s < a.tokens * a.choices; s += THREADS) {
            const int e = slot_expert(a, s);
            if (e < 0) continue;
            atomicAdd(&total[e], 1);
            if (s < first * a.choices) atomicAdd(&base[e], 1);
        }
    } else {
        // threads beside one another take neighbouring experts, groups of them every few ranges
        const int width = (a.experts + 31) / 32 * 32, step = THREADS / width, e = tid % width;
        if (e < a.experts && tid < step * width) {
            int before = 0, all = 0;
            constexpr int FLIGHT = 8;
            for (int r0 = tid / width; r0 < p.ranges; r0 += step * FLIGHT) {
                int c[FLIGHT];
#pragma unroll
                for (int f = 0; f < FLIGHT; ++f)
                    c[f] = r0 + f * step < p.ranges ? ptx::ld_dependent(p.counts + (int64_t)(r0 + f * step) * a.experts + e) : 0;
#pragma unroll
                for (int f = 0; f < FLIGHT; ++f) {
                    all += c[f];
                    before += r0 + f * step < (int)blockIdx.x ? c[f] : 0;
                }
            }
            atomicAdd(&total[e], all);
            atomicAdd(&base[e], before);
        }
    }
    __syncthreads();
    { // where each group begins: sums over the experts before it (one thread per expert)
        const int mine = tid < a.experts ? total[tid] : 0;
        int sum = warp_scan(mine);
        if (lane == 31) scan[warp] = sum;
        __syncthreads();
        if (warp == 0) scan[lane] = warp_scan(scan[lane]);
        __syncthreads();
        if (warp > 0) sum += scan[warp - 1];
        if (tid < a.experts) {
            base[tid] += sum - mine;
            if (blockIdx.x == 0) a.offsets[tid] = sum;
        }
    }

    const int tile_tokens = TILE / a.choices;
    for (int t0 = first; t0 < last; t0 += tile_tokens) {
        const int slots = (min(t0 + tile_tokens, last) - t0) * a.choices, slot = t0 * a.choices + tid;
        const int e = tid < slots ? slot_expert(a, slot) : -1;
        unsigned short *row = table + warp * pitch; // this warp's alone, until the scan below
        for (int i = lane; i < a.experts; i += 32) row[i] = 0;
        __syncwarp();
        const unsigned same = __match_any_sync(0xffffffffu, e);
        const int rank = __popc(same & ((1u << lane) - 1));
        if (e >= 0 && rank == 0) row[e] = (unsigned short)__popc(same);
        __syncthreads();
        for (int q = warp; q < a.experts; q += WARPS) { // lane = warp whose slots it counts
            const int c = table[lane * pitch + q], sum = warp_scan(c);
            table[lane * pitch + q] = (unsigned short)(sum - c);
            if (lane == 31) {
                tile_base[q] = base[q];
                base[q] += sum;
            }
        }
        __syncthreads();
        if (tid < slots) {
            const int t = slot / a.choices;
            a.positions[(int64_t)t * a.positions_ld + (slot - t * a.choices)] = e >= 0 ? tile_base[e] + row[e] + rank : -1;
        }
    }
}

// Zeros for the rows behind the last group, shared out over the grid.  E: an element.
template <typename E> __device__ __forceinline__ void zero_behind(const DispatchArgs &a, int kept) {
    char *begin = a.dst + (int64_t)max(kept, 0) * a.row_bytes, *end = a.dst + (int64_t)(a.tokens * a.choices) * a.row_bytes;
    if (begin >= end) return;
    char *low = (char *)(((uintptr_t)begin + 15) & ~(uintptr_t)15), *high = (char *)((uintptr_t)end & ~(uintptr_t)15);
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    for (char *p = low + i * 16; p < high; p += (int64_t)gridDim.x * blockDim.x * 16) *(uint4 *)p = make_uint4(0, 0, 0, 0);
    if (i < 32) { // the ends, short of a boundary (of one 16 bytes, where both lie there)
        for (char *p = begin + i * sizeof(E); p < (low < end ? low : end); p += 32 * sizeof(E)) *(E *)p = 0;
        for (char *p = (high > low ? high : low) + i * sizeof(E); p < end; p += 32 * sizeof(E)) *(E *)p = 0;
    }
}

// Both copies take the places from memory that the kernel before has written, and store only inside dst: two executions at a
// time on one scratchpad overwrite each other's counts, and the places made of them lie anywhere.
//
// Rows that start and end on 16-byte boundaries: a thread reads UNITS units of tokens' rows and stores each to its row's places.
template <int UNITS> __global__ void __launch_bounds__(256) dispatch_copy_kernel(const __grid_constant__ DispatchArgs a) {
    ptx::grid_dependency_wait();
    const int64_t units = a.row_bytes / 16, total = a.tokens * units, first = (int64_t)blockIdx.x * (256 * UNITS) + threadIdx.x;
    const uint32_t slots = (uint32_t)a.tokens * a.choices;
    uint4 v[UNITS];
    int64_t t[UNITS];
    char *dst[UNITS];
#pragma unroll
    for (int q = 0; q < UNITS; ++q) {
        const int64_t i = first + 256 * q;
        t[q] = total <= 0xffffffff ? (int64_t)((uint32_t)i / (uint32_t)units) : i / units;
        const int64_t u = i - t[q] * units;
        dst[q] = a.dst + u * 16;
        if (i < total) v[q] = ptx::ld_dependent((const uint4 *)(a.src + t[q] * a.src_pitch) + u);
        else t[q] = -1;
    }
    for (int j0 = 0; j0 < a.choices; j0 += 4) {
        int to[UNITS][4];
#pragma unroll
        for (int q = 0; q < UNITS; ++q)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                to[q][j] = j0 + j < a.choices && t[q] >= 0 ? ptx::ld_dependent(a.positions + t[q] * a.positions_ld + j0 + j) : -1;
#pragma unroll
        for (int q = 0; q < UNITS; ++q)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if ((uint32_t)to[q][j] < slots) *(uint4 *)(dst[q] + (int64_t)to[q][j] * a.row_bytes) = v[q];
    }
    zero_behind<uint32_t>(a, ptx::ld_dependent(a.offsets + a.experts - 1));
}

// Rows that start anywhere: a lane stores 16 bytes on a boundary of the place it goes to.  They come from two neighbouring
// 16-byte words of the token's row (out of L1 after the first place), shifted by the places' distance from each other's
// boundaries, which is one number for a row and a place.  E: an element.
template <typename E> __global__ void __launch_bounds__(256) dispatch_shift_kernel(const __grid_constant__ DispatchArgs a) {
    ptx::grid_dependency_wait();
    const int lane = threadIdx.x & 31;
    const uint32_t segments = (uint32_t)((a.row_bytes / 16 + 2 + 31) / 32); // 32 pieces of a row each, wherever it starts
    const int64_t item = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
    const int64_t t = item <= 0xffffffff ? (int64_t)((uint32_t)item / segments) : item / segments;
    if (t < a.tokens) {
        // offsets from the row's begin: the lane's piece, and all that may be read (a row away in either direction is enough)
        const int piece = (int)(item - t * segments) * 512 + lane * 16, bytes = (int)a.row_bytes;
        const char *row = a.src + t * a.src_pitch;
        const int low = -(int)min(t * a.src_pitch, (int64_t)bytes);
        const int high = bytes + (int)min((a.tokens - 1 - t) * a.src_pitch, (int64_t)bytes);
        const uint32_t row_at = (uint32_t)(uintptr_t)row, dst_at = (uint32_t)(uintptr_t)a.dst; // for their last four bits
        int mine = lane < a.choices ? ptx::ld_dependent(a.positions + t * a.positions_ld + lane) : -1;
        if ((uint32_t)mine >= (uint32_t)a.tokens * a.choices) mine = -1;
        for (int j = 0; j < a.choices; ++j) {
            const int to = __shfl_sync(0xffffffffu, mine, j);
            if (to < 0) continue;
            const int from = piece - (int)((dst_at + (uint32_t)to * (uint32_t)bytes) & 15);
            const int shift = (int)((row_at + (uint32_t)from) & 15), word = from - shift; // (one shift for the warp)
            char *place = a.dst + (int64_t)to * bytes;
            if (from >= 0 && from + 16 <= bytes && word >= low && word + 32 <= high) {
                const uint4 x = ptx::ld_dependent((const uint4 *)(row + word)), y = ptx::ld_dependent((const uint4 *)(row + word) + 1);
                const uint32_t w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
                uint32_t v[4];
                const int bits = (shift & 3) * 8;
                auto pick = [&](auto first) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = __funnelshift_r(w[first + i], w[first + i + 1], bits);
                };
                switch (shift >> 2) {
                    case 0: pick(std::integral_constant<int, 0>()); break;
                    case 1: pick(std::integral_constant<int, 1>()); break;
                    case 2: pick(std::integral_constant<int, 2>()); break;
                    default: pick(std::integral_constant<int, 3>()); break;
                }
                *(uint4 *)(place + from) = make_uint4(v[0], v[1], v[2], v[3]);
            } else { // the row's ends
                const int begin = max(from, 0), end = min(from + 16, bytes);
                for (int b = begin; b < end; b += sizeof(E)) *(E *)(place + b) = *(const E *)(row + b);
            }
        }
    }
    zero_behind<E>(a, ptx::ld_dependent(a.offsets + a.experts - 1));
}

// Few slots, one a thread: every CTA ranks all of them, each slot against all, and moves its share of the rows.
template <typename U, typename E> __global__ void __launch_bounds__(FEW_SLOTS) dispatch_few_kernel(const __grid_constant__ DispatchArgs a) {
    __shared__ __align__(16) int expert[FEW_SLOTS];
    __shared__ int place[FEW_SLOTS];
    __shared__ int kept;
    ptx::grid_dependency_wait();
    const int n = a.tokens * a.choices, s = threadIdx.x;
    const int64_t units = a.row_bytes / sizeof(U), work = a.tokens * units, stride = (int64_t)gridDim.x * FEW_SLOTS;
    int64_t i = (int64_t)blockIdx.x * FEW_SLOTS + s;
    const int mine = s < n ? slot_expert(a, s) : -1;
    U v;
    if (i < work) v = *((const U *)(a.src + i / units * a.src_pitch) + i % units); // on its way while the slots are ranked
    expert[s] = mine < 0 ? INT_MAX : mine; // behind all groups
    __syncthreads();
    // slots of lower experts, and of this one before; and, in the first CTA, of experts up to each
    int rank = 0;
    for (int q = 0; q < n; q += 4) {
        const int4 e = *reinterpret_cast<const int4 *>(expert + q);
        rank += (e.x < mine || (e.x == mine && q < s)) + (e.y < mine || (e.y == mine && q + 1 < s))
                + (e.z < mine || (e.z == mine && q + 2 < s)) + (e.w < mine || (e.w == mine && q + 3 < s));
    }
    place[s] = mine >= 0 ? rank : -1;
    const int there = __syncthreads_count(mine >= 0);
    if (s == 0) kept = there;
    if (blockIdx.x == 0) {
        if (s < n) a.positions[(int64_t)(s / a.choices) * a.positions_ld + s % a.choices] = place[s];
        for (int e = s; e < a.experts; e += FEW_SLOTS) {
            int ends = 0;
            for (int q = 0; q < n; q += 4) {
                const int4 x = *reinterpret_cast<const int4 *>(expert + q);
                ends += (x.x <= e) + (x.y <= e) + (x.z <= e) + (x.w <= e);
            }
            a.offsets[e] = ends;
        }
    }
    __syncthreads();
    for (; i < work; i += stride) {
        const int64_t t = i / units, u = i - t * units, next = i + stride;
        U ahead;
        if (next < work) ahead = *((const U *)(a.src + next / units * a.src_pitch) + next % units);
        for (int j = 0; j < a.choices; ++j) {
            const int to = place[t * a.choices + j];
            if (to >= 0) *((U *)(a.dst + (int64_t)to * a.row_bytes) + u) = v;
        }
        v = ahead;
    }
    zero_behind<E>(a, kept);
}

int launched(int rc) {
    if (rc == 0) count_launch();
    return rc;
}

template <typename E> int launch_copy(const DispatchArgs &a, bool aligned, cudaStream_t st) {
    if (aligned) {
        // with one place a row, more of it a thread, so that as many bytes are on their way (8192 x 4096 bf16: one choice 31.4 us
        // with one unit / 29.1 with four, two 39.2 / 39.2, four 60.6 / 61.4)
        const int units = a.choices == 1 ? 4 : 1;
        const int64_t grid = (a.tokens * (a.row_bytes / 16) + 256 * units - 1) / (256 * units);
        return grid > INT_MAX ? 3 : launched(launch_dependent(units == 4 ? dispatch_copy_kernel<4> : dispatch_copy_kernel<1>, a, (unsigned)grid, 256, 0, st));
    }
    const int64_t grid = (a.tokens * ((a.row_bytes / 16 + 2 + 31) / 32) + 7) / 8;
    return grid > INT_MAX ? 3 : launched(launch_dependent(dispatch_shift_kernel<E>, a, (unsigned)grid, 256, 0, st));
}

template <typename U, typename E> int launch_few(const DispatchArgs &a, int sm_count, cudaStream_t st) {
    const int64_t work = a.tokens * (a.row_bytes / (int64_t)sizeof(U));
    const unsigned grid = (unsigned)std::min<int64_t>(sm_count, std::max<int64_t>(1, (work + 127) / 128));
    return launched(launch_dependent(dispatch_few_kernel<U, E>, a, grid, FEW_SLOTS, 0, st));
}

} // namespace

// counts of up to `sm_count` ranges
size_t dispatch_scratch_bytes(int experts, int sm_count) { return (size_t)experts * sm_count * sizeof(int); }

int launch_dispatch(const DispatchArgs &a, int *scratch, int sm_count, cudaStream_t st) {
    if (a.tokens == 0) // no slots: the groups are empty, and say so
        return cudaMemsetAsync(a.offsets, 0, a.experts * sizeof(int), st) == cudaSuccess ? 0 : 5;
    const uint64_t places = (uint64_t)a.row_bytes | (uint64_t)(uintptr_t)a.dst | (uint64_t)(uintptr_t)a.src
            | (a.tokens > 1 ? (uint64_t)a.src_pitch : 0);
    const bool aligned = places % 16 == 0;
    if (!aligned && a.row_bytes > INT_MAX / 2) return 3;
    const int64_t slots = (int64_t)a.tokens * a.choices;
    if (few(slots, a.tokens * (a.row_bytes / (aligned ? 16 : a.element)), a.choices, aligned))
        return aligned           ? launch_few<uint4, uint32_t>(a, sm_count, st)
                : a.element == 4 ? launch_few<uint32_t, uint32_t>(a, sm_count, st)
                : a.element == 2 ? launch_few<uint16_t, uint16_t>(a, sm_count, st)
                                 : launch_few<uint8_t, uint8_t>(a, sm_count, st);
    Plan p {};
    p.a = a;
    p.counts = scratch;
    // a range is a tile, as long as there are no more of them than SMs
    p.range_tokens = std::max<int>(TILE / a.choices, (a.tokens + sm_count - 1) / sm_count);
    p.ranges = (a.tokens + p.range_tokens - 1) / p.range_tokens;
    const size_t smem = place_bytes(a.experts);
    const int most = (int)place_bytes(TOKEN_MAX_EXPERTS);
    int rc;
    if (slots <= SELF_SLOTS) {
        static std::atomic<unsigned long long> done;
        if (!opt_in_dynamic_smem(dispatch_place_kernel<true>, most, done)) return 5;
        rc = launched(launch_dependent(dispatch_place_kernel<true>, p, p.ranges, THREADS, smem, st));
    } else {
        static std::atomic<unsigned long long> done;
        if (!opt_in_dynamic_smem(dispatch_place_kernel<false>, most, done)) return 5;
        rc = launched(launch_dependent(dispatch_count_kernel, p, p.ranges, THREADS, 0, st));
        if (rc == 0) rc = launched(launch_dependent(dispatch_place_kernel<false>, p, p.ranges, THREADS, smem, st));
    }
    if (rc) return rc;
    if (a.row_bytes == 0) return 0;
    return a.element == 4 ? launch_copy<uint32_t>(a, aligned, st) : a.element == 2 ? launch_copy<uint16_t>(a, aligned, st) : launch_copy<uint8_t>(a, aligned, st);
}

} // namespace qmm

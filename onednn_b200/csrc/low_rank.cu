// Low-rank adapters of many requests beside a shared projection:
//   dst_t = base_t + scale_i (x_t down_i) up_i,  i = indices[t]; a row whose index names no adapter is base_t
// Bound by memory: of a row its src, base and dst cross it once, of an adapter its weights for each tile (from L2 but the first
// time); with ranks up to 128 there are 2 to 60 operations a byte, which mma.sync keeps up with.
//
// Rows are looked at in windows of 512; the rows of a window that share an adapter make tiles, wherever they stand.
//   Up to 1024 rows (512 from a rank of 33 on): one launch.  A cluster of CTAs takes a tile of up to 16 rows: each CTA multiplies its share of the src's columns with
//     the first factor, the sums of [rows][rank] meet in the CTAs' shared memory, and each CTA multiplies them with its share of
//     the second factor's columns.  So a single row's weights are streamed by a whole cluster.
//   More: two launches.  A CTA takes a tile of 32 rows through the first product, and the sums go to the scratchpad (4 r bytes
//     a row, which stay in L2); then a CTA takes 64 rows and a run of dst's columns through the second.  No CTA waits for another;
//     the second kernel starts as the first one's CTAs end, and finds its rows and asks for its first base and weights meanwhile
//     (777 rows of 37 adapters, in two launches, 20.1 us without, 17.4 with).
// Measured: 8192 rows, 4096 x 11008, rank 32, 16 adapters 106 to 132 us by the draw of the requests, 123 over eight draws (3.5 TB/s);
// at the draw that takes 113, 213 with 11009 columns, 179 with 4097: rows that start anywhere; 61 rows of 64 adapters,
// 4096 x 4096, rank 16 8.9 us.  The second product's kernel takes the same time without its MMAs, and with twice the bytes in flight, so that
// neither bounds it alone; its 960 CTAs are 3.2 rounds of the 296 that fit, and each finds its rows, makes its operand and fills its
// loads anew.  Deeper prefetch through shared memory (cp.async, three blocks a warp), 64 columns a warp and 256 contiguous bytes a row were slower or the same
// (119, 169, 130 us at a rank of 32; 108, 102, 118 for 106 at 16).
// Operands go from global memory to the registers of an MMA without shared memory: a lane reads 8 or 16 bytes, and which of the
// summed (or of the output's) columns these are is decided alike for both operands, so any order serves.
// The middle is a 32-bit sum.  The second product takes it as a sum of 16-bit parts, most significant first: two (what is left
// out is 2^-18 of a value), or three where dst has 32 bits and the parts are bf16 (2^-27).  f16 parts are made of values that a
// power of two brings just below the type's largest, row by row; what it divides is only the products, the base is added behind it.
#include <algorithm>

#include "launch.h"
#include "token_rows.cuh"

namespace qmm {

namespace {

constexpr int THREADS = 256, WARPS = THREADS / 32, WINDOW = 512;
constexpr int SEGMENTS = WINDOW / 32; // of a window: a warp's rows at a time

enum : int { VECTOR_OUTER = 0, VECTOR_RANK = 1, ELEMENTS = 2 }; // which neighbours of a factor a lane reads at once

struct LowRankPlan {
    LowRankArgs a;
    int64_t first_row, end_row; // of this launch
    float *middle; // [splits][end_row - first_row][16 RB], two launches
    int cluster; // CTAs of a tile, one launch
    int window_tiles; // CTAs (clusters) that take a window's tiles in turn
    int splits; // runs of src's columns, first of two launches; their sums follow one another in `middle`
    int chunks; // runs of dst's columns, second of two launches
    int down_mode, up_mode;
};

// a window's rows by adapter, in shared memory
template <int TM> struct Window {
    alignas(16) int index[WINDOW]; // of each row; `adapters` for none, -1 behind the last row
    unsigned short place[WINDOW]; // rows before it in the window with the same index
    unsigned short first[WINDOW]; // first row of each tile
    unsigned short rows[TM]; // of the tile
    alignas(8) const void *base[TM]; // where they start; behind the last, where that one does
    void *dst[TM];
    int counts[SEGMENTS]; // tiles that start in each
};

template <typename T> __device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __half>::value)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t ld_u16(const void *p) {
    unsigned short v;
    asm volatile("ld.global.u16 %0, [%1];" : "=h"(v) : "l"(p));
    return v;
}
__device__ __forceinline__ uint32_t ld_u32(const void *p) {
    uint32_t v;
    asm volatile("ld.global.u32 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
}
// a row's address, read from shared memory where it is used, so that no registers hold it
template <typename D> __device__ __forceinline__ D *ld_address(uint32_t at) {
    uint64_t v;
    asm volatile("ld.shared.u64 %0, [%1];" : "=l"(v) : "r"(at));
    return reinterpret_cast<D *>(v);
}
__device__ __forceinline__ float4 ld_cluster(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t peer_address(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t halves(uint32_t lo, uint32_t hi, bool upper) { return __byte_perm(lo, hi, upper ? 0x7632 : 0x5410); }

// Eight 16-bit values of a row from its column `col` on, of which `left` more are there; zeros behind them.  Rows that start
// anywhere: the two aligned blocks of 16 bytes that hold them, where both lie in the row, shifted; one by one at its ends.
template <bool VEC> __device__ __forceinline__ uint4 load_8(const uint16_t *at, int col, int left) {
    if constexpr (VEC) {
        return left > 0 ? ptx::ld_dependent((const uint4 *)at) : make_uint4(0, 0, 0, 0);
    } else {
        uint32_t w[8];
        if (col >= 8 && left >= 16) {
            const uint32_t off = (uint32_t)(uintptr_t)at & 15u; // bytes
            const uint4 *block = (const uint4 *)((uintptr_t)at - off);
            const uint4 x = ptx::ld_dependent(block), y = ptx::ld_dependent(block + 1);
            w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
            w[4] = y.x; w[5] = y.y; w[6] = y.z; w[7] = y.w;
#pragma unroll
            for (int i = 0; i < 6; ++i) w[i] = off & 8 ? w[i + 2] : w[i];
#pragma unroll
            for (int i = 0; i < 5; ++i) w[i] = off & 4 ? w[i + 1] : w[i];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = __byte_perm(w[i], w[i + 1], off & 2 ? 0x5432 : 0x3210);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t lo = 2 * i < left ? ld_u16(at + 2 * i) : 0u, hi = 2 * i + 1 < left ? ld_u16(at + 2 * i + 1) : 0u;
                w[i] = lo | hi << 16;
            }
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// The first factor's operand of 32 columns of src, of which this lane has eight: w[j] = (pairs of) those of column n(j0 + j, lane / 4)
// of the rank, where n(j, g) is 8 j + g, or 2 RB g + j where neighbours are read along the rank.  at: where the lane's first column
// meets n(0, g); left: columns of src from there on.
template <int RB, int J, bool VEC>
__device__ __forceinline__ void load_down(uint32_t (&w)[J][4], const LowRankPlan &p, const uint16_t *at, int left, int j0, int lane) {
    const LowRankArgs &a = p.a;
    const int g = lane >> 2;
    if (p.down_mode == VECTOR_OUTER) {
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const uint4 v = 8 * (j0 + j) + g < a.rank && left > 0 ? ptx::ld_dependent((const uint4 *)(at + 8 * (j0 + j) * a.down_rank)) : make_uint4(0, 0, 0, 0);
            w[j][0] = v.x; w[j][1] = v.y; w[j][2] = v.z; w[j][3] = v.w;
        }
    } else if (VEC || p.down_mode == VECTOR_RANK) {
        uint32_t rows[8][J / 2]; // two columns of the rank a word
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const bool there = 2 * RB * g < a.rank && i < left;
            const uint16_t *from = at + i * a.down_in + j0;
#pragma unroll
            for (int q = 0; q < J / 2; ++q) rows[i][q] = 0;
            if (there) {
                if constexpr (J == 2) rows[i][0] = ld_u32(from);
                else if constexpr (J == 4) {
                    const uint2 v = ptx::ld_dependent((const uint2 *)from);
                    rows[i][0] = v.x; rows[i][1] = v.y;
                } else {
                    const uint4 v = ptx::ld_dependent((const uint4 *)from);
                    rows[i][0] = v.x; rows[i][1] = v.y; rows[i][2] = v.z; rows[i][3] = v.w;
                }
            }
        }
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) w[j][i] = halves(rows[2 * i][j / 2], rows[2 * i + 1][j / 2], j & 1);
    } else {
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const bool there = 8 * (j0 + j) + g < a.rank;
            if (a.down_in == 1) { // rows that start anywhere
                const uint4 v = load_8<false>(at + 8 * (j0 + j) * a.down_rank, (int)a.in - left, there ? left : 0);
                w[j][0] = v.x; w[j][1] = v.y; w[j][2] = v.z; w[j][3] = v.w;
                continue;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint16_t *from = at + 8 * (j0 + j) * a.down_rank + 2 * i * a.down_in;
                const uint32_t lo = there && 2 * i < left ? ld_u16(from) : 0u;
                const uint32_t hi = there && 2 * i + 1 < left ? ld_u16(from + a.down_in) : 0u;
                w[j][i] = lo | hi << 16;
            }
        }
    }
}

// column of the rank that value i (of four) of a lane is, in the second product's step s
template <int RB> __device__ __forceinline__ int rank_column(int mode, int s, int t, int i) {
    return mode == VECTOR_RANK ? t * 4 * RB + 4 * s + i : 16 * s + 4 * t + i;
}

// The second factor's operand of 32 columns of dst: w[j][s] = this lane's four values of the rank in step s at column
// 4 (lane / 4) + j.  (So a lane ends up with eight neighbours of a row of dst: columns 2 t and 2 t + 1 of the four products.)
// It is loaded as it lies in memory, and brought into this order where it is used.  at: where the lane's first column meets its
// first value of the rank; left: columns of dst from there on.
template <int RB, bool VEC>
__device__ __forceinline__ void load_up(uint32_t (&w)[8 * RB], const LowRankPlan &p, const uint16_t *at, int left, int lane) {
    const LowRankArgs &a = p.a;
    const int t = lane & 3;
    if (p.up_mode == VECTOR_OUTER) { // [value of the rank][pair of columns]
#pragma unroll
        for (int s = 0; s < RB; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint2 v = 16 * s + 4 * t + i < a.rank && left > 0 ? ptx::ld_dependent((const uint2 *)(at + (16 * s + i) * a.up_rank)) : make_uint2(0, 0);
                w[8 * s + 2 * i] = v.x; w[8 * s + 2 * i + 1] = v.y;
            }
    } else if (VEC || p.up_mode == VECTOR_RANK) { // [column][pair of the rank]
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bool there = j < left && t * 4 * RB < a.rank;
            const uint16_t *from = at + j * a.up_out;
            if constexpr (RB == 1) {
                const uint2 v = there ? ptx::ld_dependent((const uint2 *)from) : make_uint2(0, 0);
                w[2 * j] = v.x; w[2 * j + 1] = v.y;
            } else {
#pragma unroll
                for (int s = 0; s < RB; s += 2) {
                    const uint4 v = there ? ptx::ld_dependent((const uint4 *)(from + 4 * s)) : make_uint4(0, 0, 0, 0);
                    w[2 * RB * j + 2 * s] = v.x; w[2 * RB * j + 2 * s + 1] = v.y;
                    w[2 * RB * j + 2 * s + 2] = v.z; w[2 * RB * j + 2 * s + 3] = v.w;
                }
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int q = 0; q < 2 * RB; ++q) {
                const int k = 16 * (q / 2) + 2 * (q % 2);
                const uint16_t *from = at + j * a.up_out + k * a.up_rank;
                const uint32_t lo = j < left && 4 * t + k < a.rank ? ld_u16(from) : 0u;
                const uint32_t hi = j < left && 4 * t + k + 1 < a.rank ? ld_u16(from + a.up_rank) : 0u;
                w[2 * RB * j + q] = lo | hi << 16;
            }
    }
}
template <int RB> __device__ __forceinline__ void order_up(uint32_t (&w)[4][RB][2], const uint32_t (&raw)[8 * RB], const LowRankPlan &p) {
    if (p.up_mode == VECTOR_OUTER) {
#pragma unroll
        for (int s = 0; s < RB; ++s)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j][s][h] = halves(raw[8 * s + 4 * h + j / 2], raw[8 * s + 4 * h + 2 + j / 2], j & 1);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int q = 0; q < 2 * RB; ++q) w[j][q / 2][q % 2] = raw[2 * RB * j + q];
    }
}

// eight values of a row of base or dst from its column `col` on, of which `left` more are there
template <typename D, bool VEC> struct Eight {
    uint4 raw[sizeof(D) / 2];
    __device__ __forceinline__ void load(const D *at, int col, int left) {
        if constexpr (sizeof(D) == 2) {
            raw[0] = load_8<VEC>((const uint16_t *)at, col, left);
        } else if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < 2; ++i) raw[i] = left > 0 ? ptx::ld_dependent((const uint4 *)at + i) : make_uint4(0, 0, 0, 0);
        } else {
            uint32_t w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = i < left ? ld_u32(at + i) : 0u;
            raw[0] = make_uint4(w[0], w[1], w[2], w[3]);
            raw[1] = make_uint4(w[4], w[5], w[6], w[7]);
        }
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        if constexpr (sizeof(D) == 4) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                v[4 * i] = __uint_as_float(raw[i].x);
                v[4 * i + 1] = __uint_as_float(raw[i].y);
                v[4 * i + 2] = __uint_as_float(raw[i].z);
                v[4 * i + 3] = __uint_as_float(raw[i].w);
            }
        } else {
            unpack2(raw[0].x, v[0], v[1], D());
            unpack2(raw[0].y, v[2], v[3], D());
            unpack2(raw[0].z, v[4], v[5], D());
            unpack2(raw[0].w, v[6], v[7], D());
        }
    }
    static __device__ __forceinline__ void store_pair(D *at, float lo, float hi) {
        if constexpr (sizeof(D) == 2) *reinterpret_cast<uint32_t *>(at) = pack2(lo, hi, D());
    }
    static __device__ __forceinline__ void store(D *at, int left, const float (&v)[8]) {
        if constexpr (VEC) {
            if (left > 0) Cols<D, true>::store_ragged(at, 8, v);
        } else if (sizeof(D) == 2 && left >= 8) { // in words of two, where they are aligned
            const bool odd = (uintptr_t)at & 2;
            if (odd) {
                at[0] = from_f32<D>(v[0]);
                at[7] = from_f32<D>(v[7]);
#pragma unroll
                for (int i = 1; i < 7; i += 2) store_pair(at + i, v[i], v[i + 1]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; i += 2) store_pair(at + i, v[i], v[i + 1]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < left) at[i] = from_f32<D>(v[i]);
        }
    }
};

// The sums of this warp's share of the src's columns, U steps of 32 at a time, for the tile's M groups of 16 rows.
template <typename T, int RB, bool VEC, int M, int U>
__device__ __forceinline__ void first_product(float (&acc)[M][2 * RB][4], const LowRankPlan &p, const uint16_t *down, const unsigned short *rows,
        int64_t window, int count, int lane, int first, int step) {
    const LowRankArgs &a = p.a;
    constexpr int J = 2 * RB < 8 ? 2 * RB : 8; // blocks of eight of the rank at a time
    const int g = lane >> 2, t = lane & 3;
    const uint16_t *x[M][2]; // rows g and g + 8 of a group
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h)
            x[m][h] = (const uint16_t *)a.src + (window + rows[min(16 * m + 8 * h + g, count - 1)]) * a.src_ld + 32 * first + 8 * t;
    down += p.down_mode == VECTOR_RANK ? 2 * RB * g : g * a.down_rank;
    int left = (int)a.in - 32 * first - 8 * t;
    for (int s = first; 32 * s < (int)a.in; s += U * step) {
        uint32_t w[U][J][4];
        uint4 v[U][M][2];
#pragma unroll
        for (int u = 0; u < U; ++u) { // (steps behind the last read zeros)
#pragma unroll
            for (int m = 0; m < M; ++m)
#pragma unroll
                for (int h = 0; h < 2; ++h) v[u][m][h] = load_8<VEC>(x[m][h] + 32 * u * step, (int)a.in - left + 32 * u * step, left - 32 * u * step);
            load_down<RB, J, VEC>(w[u], p, down + (32 * (s + u * step) + 8 * t) * a.down_in, left - 32 * u * step, 0, lane);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j0 = 0; j0 < 2 * RB; j0 += J) {
                if (j0 > 0) load_down<RB, J, VEC>(w[u], p, down + (32 * (s + u * step) + 8 * t) * a.down_in, left - 32 * u * step, j0, lane);
#pragma unroll
                for (int m = 0; m < M; ++m)
#pragma unroll
                    for (int j = 0; j < J; ++j) {
                        mma_16816<T>(acc[m][j0 + j], v[u][m][0].x, v[u][m][1].x, v[u][m][0].y, v[u][m][1].y, w[u][j][0], w[u][j][1]);
                        mma_16816<T>(acc[m][j0 + j], v[u][m][0].z, v[u][m][1].z, v[u][m][0].w, v[u][m][1].w, w[u][j][2], w[u][j][3]);
                    }
            }
        left -= 32 * U * step;
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h) x[m][h] += 32 * U * step;
    }
}

// Fills in `sh` from the indices of the window's rows; returns the number of its tiles.  counts: sixteen bytes for every adapter
// and for none, of shared memory that is free until the next barrier.
template <int TM> __device__ __forceinline__ int find_tiles(Window<TM> &sh, uint4 *counts, const LowRankArgs &a, int64_t window, int rows) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    for (int i = threadIdx.x; i <= a.adapters; i += THREADS) counts[i] = make_uint4(0, 0, 0, 0);
    int ids[2]; // of rows threadIdx.x and THREADS + threadIdx.x
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int i = h * THREADS + threadIdx.x;
        ids[h] = -1;
        if (i < rows) {
            ids[h] = ptx::ld_dependent(a.indices + window + i);
            if ((unsigned)ids[h] >= (unsigned)a.adapters) ids[h] = a.adapters;
        }
        sh.index[i] = ids[h];
    }
    __syncthreads();
    uint32_t same[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) { // [adapter][segment]: rows of the segment with this index
        same[h] = __match_any_sync(0xffffffffu, ids[h]);
        if (ids[h] >= 0 && lane == __ffs(same[h]) - 1)
            reinterpret_cast<unsigned char *>(counts + ids[h])[h * WARPS + warp] = (unsigned char)__popc(same[h]);
    }
    __syncthreads();
    bool leads[2]; // a row that has a multiple of TM rows of its index before it is the first of a tile
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int i = h * THREADS + threadIdx.x, segment = h * WARPS + warp;
        int before = __popc(same[h] & ((1u << lane) - 1));
        if (ids[h] >= 0) {
            const uint4 v = counts[ids[h]];
            const uint32_t word[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int q = 0; q < 4; ++q) { // bytes of the segments before this one
                const int bytes = min(max(segment - 4 * q, 0), 4);
                before = __dp4a(word[q] & (uint32_t)((1ull << 8 * bytes) - 1), 0x01010101u, (uint32_t)before);
            }
        }
        sh.place[i] = (unsigned short)before;
        leads[h] = ids[h] >= 0 && before % TM == 0;
        const uint32_t firsts = __ballot_sync(0xffffffffu, leads[h]);
        if (lane == 0) sh.counts[segment] = __popc(firsts);
    }
    __syncthreads();
    const int mine = lane < SEGMENTS ? sh.counts[lane] : 0;
    int through = mine; // tiles that start in the segments up to `lane`
#pragma unroll
    for (int s = 1; s < SEGMENTS; s *= 2) {
        const int v = __shfl_up_sync(0xffffffffu, through, s);
        if (lane >= s) through += v;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int at = __shfl_sync(0xffffffffu, through - mine, h * WARPS + warp);
        const uint32_t firsts = __ballot_sync(0xffffffffu, leads[h]);
        if (leads[h]) sh.first[at + __popc(firsts & ((1u << lane) - 1))] = (unsigned short)(h * THREADS + threadIdx.x);
    }
    return __shfl_sync(0xffffffffu, through, SEGMENTS - 1);
}

// Adapter and rows (sh.rows, `count` of them) of a tile; barriers before and behind.
template <int TM> __device__ __forceinline__ int find_rows(Window<TM> &sh, int tile, int &count) {
    __syncthreads();
    const int lead = sh.first[tile], id = sh.index[lead], first = sh.place[lead];
    count = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int i = h * THREADS + threadIdx.x, at = sh.place[i] - first;
        const bool mine = sh.index[i] == id && at >= 0 && at < TM;
        if (mine) sh.rows[at] = (unsigned short)i;
        count += __syncthreads_count(mine);
    }
    return id;
}
// where the tile's rows of base and dst start; read behind the next barrier
template <typename D, int TM> __device__ __forceinline__ void find_addresses(Window<TM> &sh, const LowRankArgs &a, int64_t window, int count) {
    if (threadIdx.x < TM) {
        const int64_t row = window + sh.rows[min((int)threadIdx.x, count - 1)];
        sh.base[threadIdx.x] = (const D *)a.base + row * a.base_ld;
        sh.dst[threadIdx.x] = (D *)a.dst + row * a.dst_ld;
    }
}

// dst = base in blocks of 32 columns, for rows without an adapter
template <typename D, bool VEC>
__device__ __forceinline__ void copy_rows(const LowRankArgs &a, const unsigned short *rows, int64_t window, int count, int first_block, int end_block) {
    if (a.base == a.dst && a.base_ld == a.dst_ld) return; // in place
    const int lane = threadIdx.x & 31;
    for (int b = first_block; b < end_block; b += WARPS) {
        const int col = 32 * b + 8 * (lane & 3), left = (int)a.out - col;
        for (int r = lane >> 2; r < count; r += 8) {
            const int64_t row = window + rows[r];
            float v[8] = {};
            if (a.base) {
                Eight<D, VEC> e;
                e.load((const D *)a.base + row * a.base_ld + col, col, left);
                e.get(v);
            }
            Eight<D, VEC>::store((D *)a.dst + row * a.dst_ld + col, left, v);
        }
    }
}

// Sums of the warps, [rows][rank]: the upper four warps' sums to shared memory, the lower four's on top of them; what is left is four slabs.
template <int RB, int M> struct Slabs {
    static constexpr int PITCH = 16 * RB + 4;
    float v[WARPS / 2][16 * M][PITCH];
    __device__ __forceinline__ void add(const float (&acc)[M][2 * RB][4], int down_mode) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
#pragma unroll
        for (int round = 0; round < 2; ++round) {
            if ((warp < WARPS / 2) == (round == 1)) {
#pragma unroll
                for (int m = 0; m < M; ++m)
#pragma unroll
                    for (int j = 0; j < 2 * RB; ++j)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int c = 2 * (lane & 3) + i % 2, col = down_mode == VECTOR_RANK ? 2 * RB * c + j : 8 * j + c;
                            float *at = &v[warp % (WARPS / 2)][16 * m + 8 * (i / 2) + (lane >> 2)][col];
                            *at = round ? acc[m][j][i] + *at : acc[m][j][i];
                        }
            }
            __syncthreads();
        }
    }
    __device__ __forceinline__ float sum(int row, int col) const {
        return (v[0][row][col] + v[1][row][col]) + (v[2][row][col] + v[3][row][col]);
    }
};

template <typename T, typename D> constexpr int PARTS = sizeof(D) == 4 && std::is_same<T, __nv_bfloat16>::value ? 3 : 2;

// The second product's left operand, for a row of which this thread (of four, t = threadIdx.x % 4) has the middle's columns
// rank_column(mode, s, t, 0..3): operand[part][group of rows][s][lane].  f16: returns the power of two it was divided by.
template <typename T, int RB, int P>
__device__ __forceinline__ float make_operand(uint4 *operand, int groups, float (&v)[RB][4], const LowRankPlan &p, int row, bool there) {
    const int t = threadIdx.x % 4;
    float most = 0.f, unit = 1.f;
#pragma unroll
    for (int s = 0; s < RB; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (rank_column<RB>(p.up_mode, s, t, i) >= p.a.rank) v[s][i] = 0.f; // (whatever src holds)
            most = fmaxf(most, fabsf(v[s][i]));
        }
    if constexpr (std::is_same<T, __half>::value) { // the largest of the row into [2^13, 2^14), by a normal number
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        if (most > 0.f && most < INFINITY) unit = __uint_as_float(max(__float_as_uint(most) & 0x7f800000u, 14u << 23)) * 0x1p-13f;
    }
    if (!there) return unit;
    const float inverse = 1.f / unit;
    const int at = (row / 16 * RB) * 32 + row % 8 * 4 + t, word = row % 16 / 8;
#pragma unroll
    for (int s = 0; s < RB; ++s) {
        float rest[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) rest[i] = v[s][i] * inverse;
#pragma unroll
        for (int q = 0; q < P; ++q) {
            uint32_t *to = reinterpret_cast<uint32_t *>(operand + (q * groups * RB + s) * 32 + at) + word;
            alignas(8) T part[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                part[i] = from_f32<T>(rest[i]);
                const float left = rest[i] - to_f32(part[i]);
                rest[i] = fabsf(to_f32(part[i])) < INFINITY ? left : 0.f;
            }
            to[0] = reinterpret_cast<const uint32_t *>(part)[0];
            to[2] = reinterpret_cast<const uint32_t *>(part)[1];
        }
    }
    return unit;
}

// Second product of the tile's GROUPS groups of 16 rows, from the operand in shared memory.  A warp has M of them and works on 32
// columns of dst at a time, every `stride` of these blocks; its rows' base is asked for one block ahead, the weights too where
// registers allow it (a rank of up to 32).  start() asks for the first block's, and may be called long before.
template <typename T, typename D, int RB, bool VEC, int M, int GROUPS> struct SecondProduct {
    static constexpr bool AHEAD = RB <= 2, UNITS = std::is_same<T, __half>::value;
    // With units the next base can be asked for behind the products only; the weights in front of it where registers allow it (8192 rows of
    // 37 adapters, 2048 x 5504, f16, us a call, in front / behind: rank 64 to f32 250 / 280; to f16, 16 adapters 4096 x 11008, 192 / 181;
    // rank 128 to f32 433 / 426).
    static constexpr bool WEIGHTS_FIRST = UNITS && RB == 4 && sizeof(D) == 4;
    const LowRankPlan &p;
    const uint16_t *up; // of the lane, in the block that is asked for next
    uint32_t bases, dsts; // shared memory, of the lane's first row
    int count, lane, group, end, stride;
    uint32_t raw[8 * RB];
    Eight<D, VEC> base[M][2];

    // group: the warp's first; blocks first, first + stride, ... below end
    __device__ __forceinline__ SecondProduct(const LowRankPlan &p, const uint16_t *up, const Window<16 * GROUPS> &rows, int count, int lane,
            int group, int first, int end, int stride)
        : p(p), count(count), lane(lane), group(group), end(end), stride(stride) {
        bases = ptx::smem_u32(rows.base + 16 * group + (lane >> 2));
        dsts = ptx::smem_u32(rows.dst + 16 * group + (lane >> 2));
        this->up = up + (32 * first + 4 * (lane >> 2)) * p.a.up_out + rank_column<RB>(p.up_mode, 0, lane & 3, 0) * p.a.up_rank;
    }
    __device__ __forceinline__ void load_base(int m, int h, int col) {
        base[m][h].load(ld_address<const D>(bases + 8 * (16 * m + 8 * h)) + col, col, (int)p.a.out - col);
    }
    __device__ __forceinline__ void load_weights(int b) {
        load_up<RB, VEC>(raw, p, up, (int)p.a.out - 32 * b - 4 * (lane >> 2), lane);
        up += 32 * stride * p.a.up_out;
    }
    __device__ __forceinline__ void start(int first) {
        if (first >= end) return;
        if (p.a.base) {
#pragma unroll
            for (int m = 0; m < M; ++m)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    if (16 * (group + m) < count) load_base(m, h, 32 * first + 8 * (lane & 3));
        }
        load_weights(first);
    }
    __device__ __forceinline__ void run(int first, const uint4 *operand, const float *units) {
        for (int b = first; b < end; b += stride) {
            const int col = 32 * b + 8 * (lane & 3);
            const bool more = b + stride < end;
            uint32_t w[4][RB][2];
            order_up<RB>(w, raw, p);
            if (AHEAD && more) load_weights(b + stride);
#pragma unroll
            for (int m = 0; m < M; ++m) {
                if (16 * (group + m) >= count) break;
                // The base is where the sums begin (bf16), or is added to them behind their unit (f16: in that unit a finite base might be infinite).
                float out[4][4];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float v[8] = {};
                    if (!UNITS && p.a.base) {
                        base[m][h].get(v);
                        if (more) load_base(m, h, col + 32 * stride);
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int i = 0; i < 2; ++i) out[j][2 * h + i] = v[4 * i + j];
                }
#pragma unroll
                for (int q = PARTS<T, D> - 1; q >= 0; --q) // the smallest first
#pragma unroll
                    for (int s = 0; s < RB; ++s) {
                        const uint4 f = operand[((q * GROUPS + group + m) * RB + s) * 32 + lane];
#pragma unroll
                        for (int j = 0; j < 4; ++j) mma_16816<T>(out[j], f.x, f.y, f.z, f.w, w[j][s][0], w[j][s][1]);
                    }
                if (WEIGHTS_FIRST && more && (m == M - 1 || 16 * (group + m + 1) >= count)) load_weights(b + stride);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float v[8] = {};
                    if (UNITS && p.a.base) {
                        base[m][h].get(v);
                        if (more) load_base(m, h, col + 32 * stride);
                    }
                    const float unit = UNITS ? units[16 * (group + m) + 8 * h + (lane >> 2)] : 1.f;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int i = 0; i < 2; ++i) v[4 * i + j] = UNITS ? fmaf(out[j][2 * h + i], unit, v[4 * i + j]) : out[j][2 * h + i];
                    if (16 * (group + m) + 8 * h + (lane >> 2) < count)
                        Eight<D, VEC>::store(ld_address<D>(dsts + 8 * (16 * m + 8 * h)) + col, (int)p.a.out - col, v);
                }
            }
            if (!AHEAD && !WEIGHTS_FIRST && more) load_weights(b + stride);
        }
    }
};

// ------------------------------------------------------------------------------------------------- one launch

template <typename T, typename D, int RB> struct FewShared {
    union {
        uint4 counts[LOW_RANK_MAX_ADAPTERS + 1];
        Slabs<RB, 1> slabs;
        uint4 operand[PARTS<T, D> * RB * 32];
    };
    alignas(16) float part[16][16 * RB]; // this CTA's sums, which the whole cluster reads
    float unit[16];
    Window<16> window;
};

template <typename T, typename D, int RB, bool VEC>
__global__ void __launch_bounds__(THREADS) low_rank_few_kernel(const __grid_constant__ LowRankPlan p) {
    __shared__ FewShared<T, D, RB> sh;
    ptx::grid_dependency_wait();
    const LowRankArgs &a = p.a;
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32, rank = (int)cluster_rank();
    const int number = (int)blockIdx.x / p.cluster; // of the cluster
    const int64_t window = p.first_row + (int64_t)(number / p.window_tiles) * WINDOW;
    const int tiles = find_tiles(sh.window, sh.counts, a, window, (int)min((int64_t)WINDOW, p.end_row - window));
    const int64_t blocks = (a.out + 31) / 32; // of 32 columns of dst, in runs of neighbours for each CTA
    const int first = (int)(blocks * rank / p.cluster) + warp, end = (int)(blocks * (rank + 1) / p.cluster);
    bool arrived = false; // at the barrier behind the reads of `part`
    for (int tile = number % p.window_tiles; tile < tiles; tile += p.window_tiles) {
        int count;
        const int id = find_rows(sh.window, tile, count);
        if (id == a.adapters) {
            copy_rows<D, VEC>(a, sh.window.rows, window, count, first, end);
            continue;
        }
        find_addresses<D>(sh.window, a, window, count);
        float acc[1][2 * RB][4] = {};
        first_product<T, RB, VEC, 1, (RB > 2 ? 1 : (VEC ? 4 : 2) / RB)>(acc, p, (const uint16_t *)a.down + id * a.down_adapter, sh.window.rows,
                window, count, lane, rank * WARPS + warp, p.cluster * WARPS);
        __syncthreads();
        SecondProduct<T, D, RB, VEC, 1, 1> second(p, (const uint16_t *)a.up + id * a.up_adapter, sh.window, count, lane, 0, first, end, WARPS);
        second.start(first); // on its way meanwhile
        sh.slabs.add(acc, p.down_mode);
        if (arrived) cluster_wait(); // (the last tile's `part` has been read everywhere)
        for (int i = threadIdx.x; i < 16 * 16 * RB; i += THREADS) sh.part[i / (16 * RB)][i % (16 * RB)] = sh.slabs.sum(i / (16 * RB), i % (16 * RB));
        cluster_arrive();
        cluster_wait();
        if (threadIdx.x < 64) {
            const int row = threadIdx.x / 4;
            const float scale = a.scales ? ptx::ld_dependent(a.scales + id) : 1.f;
            float v[RB][4];
#pragma unroll
            for (int s = 0; s < RB; ++s) {
                const uint32_t at = ptx::smem_u32(&sh.part[row][rank_column<RB>(p.up_mode, s, threadIdx.x % 4, 0)]);
                float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
                for (int c = 0; c < p.cluster; ++c) {
                    const float4 q = ld_cluster(peer_address(at, c));
                    sum.x += q.x; sum.y += q.y; sum.z += q.z; sum.w += q.w;
                }
                v[s][0] = sum.x * scale; v[s][1] = sum.y * scale; v[s][2] = sum.z * scale; v[s][3] = sum.w * scale;
            }
            const float unit = make_operand<T, RB, PARTS<T, D>>(sh.operand, 1, v, p, row, true);
            if (threadIdx.x % 4 == 0) sh.unit[row] = unit;
        }
        cluster_arrive();
        arrived = true;
        __syncthreads();
        second.run(first, sh.operand, sh.unit);
    }
    if (arrived) cluster_wait(); // nobody leaves while its sums may be read
}

// ------------------------------------------------------------------------------------------------ two launches

template <int RB> constexpr int DOWN_GROUPS = RB == 8 ? 1 : 2; // of 16 rows

template <typename T, int RB, bool VEC>
__global__ void __launch_bounds__(THREADS, RB <= 2 ? 2 : 1) low_rank_down_kernel(const __grid_constant__ LowRankPlan p) {
    constexpr int M = DOWN_GROUPS<RB>;
    __shared__ union {
        uint4 counts[LOW_RANK_MAX_ADAPTERS + 1];
        Slabs<RB, M> slabs;
    } sh;
    __shared__ Window<16 * M> rows;
    ptx::grid_dependency_wait();
    asm volatile("griddepcontrol.launch_dependents;"); // (the second product's CTAs read the sums behind their own wait)
    const LowRankArgs &a = p.a;
    const int split = (int)blockIdx.x % p.splits, number = (int)blockIdx.x / p.splits;
    const int64_t window = p.first_row + (int64_t)(number / p.window_tiles) * WINDOW;
    float *middle = p.middle + split * (p.end_row - p.first_row) * (16 * RB);
    const int tiles = find_tiles(rows, sh.counts, a, window, (int)min((int64_t)WINDOW, p.end_row - window));
    for (int tile = number % p.window_tiles; tile < tiles; tile += p.window_tiles) {
        int count;
        const int id = find_rows(rows, tile, count);
        if (id == a.adapters) continue;
        float acc[M][2 * RB][4] = {};
        first_product<T, RB, VEC, M, (!VEC || RB > 2 ? 1 : 2)>(acc, p, (const uint16_t *)a.down + id * a.down_adapter, rows.rows, window, count,
                threadIdx.x & 31, split * WARPS + threadIdx.x / 32, p.splits * WARPS);
        sh.slabs.add(acc, p.down_mode);
        const float scale = a.scales ? ptx::ld_dependent(a.scales + id) : 1.f;
        for (int i = threadIdx.x; i < count * 16 * RB; i += THREADS) {
            const int row = i / (16 * RB), col = i % (16 * RB);
            middle[(window - p.first_row + rows.rows[row]) * (16 * RB) + col] = sh.slabs.sum(row, col) * scale;
        }
    }
}

template <typename D, int RB> constexpr int UP_GROUPS = sizeof(D) == 2 && RB <= 2 ? 4 : 2; // of 16 rows, of a warp
template <int RB> constexpr int UP_CTAS = RB <= 4 ? 2 : 1; // of an SM

template <typename T, typename D, int RB> struct UpShared {
    union {
        uint4 counts[LOW_RANK_MAX_ADAPTERS + 1];
        uint4 operand[PARTS<T, D> * 4 * RB * 32];
    };
    float unit[64];
    Window<64> window;
};

template <typename T, typename D, int RB, bool VEC>
__global__ void __launch_bounds__(THREADS, UP_CTAS<RB>) low_rank_up_kernel(const __grid_constant__ LowRankPlan p) {
    extern __shared__ __align__(16) unsigned char shared[];
    UpShared<T, D, RB> &sh = *reinterpret_cast<UpShared<T, D, RB> *>(shared);
    // What this kernel reads before it waits for the first product's end - indices, base, weights - the first product's kernel has
    // waited for: all its CTAs had done so when this one could start.
    const LowRankArgs &a = p.a;
    bool waited = false;
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    const int chunk = (int)blockIdx.x % p.chunks, number = (int)blockIdx.x / p.chunks;
    const int64_t window = p.first_row + (int64_t)(number / p.window_tiles) * WINDOW;
    const int tiles = find_tiles(sh.window, sh.counts, a, window, (int)min((int64_t)WINDOW, p.end_row - window));
    const int64_t blocks = (a.out + 31) / 32;
    const int begin = (int)(blocks * chunk / p.chunks), end = (int)(blocks * (chunk + 1) / p.chunks);
    for (int tile = number % p.window_tiles; tile < tiles; tile += p.window_tiles) {
        int count;
        const int id = find_rows(sh.window, tile, count);
        if (id == a.adapters) {
            if (!waited) ptx::grid_dependency_wait(); // (whoever reads dst's memory before has ended)
            waited = true;
            copy_rows<D, VEC>(a, sh.window.rows, window, count, begin + warp, end);
            continue;
        }
        find_addresses<D>(sh.window, a, window, count);
        __syncthreads();
        // Where a warp's rows are fewer than the tile's, neighbouring warps share the columns.
        constexpr int M = UP_GROUPS<D, RB>;
        const int parts = 16 * M < count ? 4 / M : 1, first = begin + warp / parts;
        SecondProduct<T, D, RB, VEC, M, 4> second(p, (const uint16_t *)a.up + id * a.up_adapter, sh.window, count, lane, warp % parts * M, first,
                end, WARPS / parts);
        second.start(first);
        if (!waited) ptx::grid_dependency_wait();
        waited = true;
        const int row = threadIdx.x / 4;
        float v[RB][4] = {};
        if (row < count) {
            const float *middle = p.middle + (window - p.first_row + sh.window.rows[row]) * (16 * RB);
            for (int split = 0; split < p.splits; ++split, middle += (p.end_row - p.first_row) * (16 * RB))
#pragma unroll
                for (int s = 0; s < RB; ++s) {
                    const float4 q = ptx::ld_dependent((const float4 *)(middle + rank_column<RB>(p.up_mode, s, threadIdx.x % 4, 0)));
                    v[s][0] += q.x; v[s][1] += q.y; v[s][2] += q.z; v[s][3] += q.w;
                }
        }
        const float unit = make_operand<T, RB, PARTS<T, D>>(sh.operand, 4, v, p, row, row < (count + 15) / 16 * 16);
        if (threadIdx.x % 4 == 0) sh.unit[row] = unit;
        __syncthreads();
        second.run(first, sh.operand, sh.unit);
    }
    if (!waited) ptx::grid_dependency_wait(); // (the next kernel on the stream relies on this one's wait)
}

template <typename Kernel> int launch_cluster(Kernel kernel, const LowRankPlan &p, unsigned grid, cudaStream_t st) {
    cudaLaunchConfig_t cfg {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(THREADS);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = p.cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    void *kargs[] = {const_cast<LowRankPlan *>(&p)};
    const int rc = cudaLaunchKernelExC(&cfg, (const void *)kernel, kargs) == cudaSuccess ? 0 : 5;
    if (rc == 0) count_launch();
    return rc;
}

template <typename T, typename D, int RB, bool VEC> int launch_few(LowRankPlan &p, int sm_count, cudaStream_t st) {
    const LowRankArgs &a = p.a;
    const int64_t windows = (a.rows + WINDOW - 1) / WINDOW, most = std::min<int64_t>(a.rows, WINDOW);
    p.end_row = a.rows;
    p.cluster = 4;
    p.window_tiles = (int)std::min<int64_t>(most, std::max<int64_t>(WINDOW / 16 + 2, 2 * sm_count / (windows * p.cluster)));
    return launch_cluster(low_rank_few_kernel<T, D, RB, VEC>, p, (unsigned)(windows * p.window_tiles * p.cluster), st);
}

template <typename T, typename D, int RB> int launch_many(LowRankPlan &p, bool in, bool out, int sm_count, cudaStream_t st) {
    const LowRankArgs &a = p.a;
    static std::atomic<unsigned long long> done, done_any;
    if (!opt_in_dynamic_smem(low_rank_up_kernel<T, D, RB, true>, (int)sizeof(UpShared<T, D, RB>), done)
            || !opt_in_dynamic_smem(low_rank_up_kernel<T, D, RB, false>, (int)sizeof(UpShared<T, D, RB>), done_any))
        return 5;
    for (p.first_row = 0; p.first_row < a.rows; p.first_row = p.end_row) {
        p.end_row = std::min<int64_t>(a.rows, p.first_row + LOW_RANK_CHUNK);
        const int64_t rows = p.end_row - p.first_row, windows = (rows + WINDOW - 1) / WINDOW, most = std::min<int64_t>(rows, WINDOW);
        // Full tiles, and half of the adapters once more a window.  The columns of src are split where tiles are too few for the SMs
        // (us a call, one / two / four splits: 777 rows, 37 adapters, 2048 x 5504, in two launches, 23.2 / 21.0 / 21.7; 8192 rows,
        // 16 adapters, 4096 x 11008, one draw of requests, 118.4 / 118.2 / 122.9).
        const int64_t ends = windows * (std::min<int64_t>(most, a.adapters) / 2 + 1);
        p.splits = (int)std::min<int64_t>(LOW_RANK_SPLITS, std::max<int64_t>(1, sm_count / (ends + rows / (16 * DOWN_GROUPS<RB>))));
        p.window_tiles = (int)std::min<int64_t>(most, std::max<int64_t>(WINDOW / (16 * DOWN_GROUPS<RB>) + 2, 2 * sm_count / (windows * p.splits)));
        int rc = launch_dependent(in ? low_rank_down_kernel<T, RB, true> : low_rank_down_kernel<T, RB, false>, p,
                (unsigned)(windows * p.window_tiles * p.splits), THREADS, 0, st);
        if (rc != 0) return rc;
        count_launch();
        // Three rounds of CTAs, of at least three blocks of columns a warp (us a call, four / six / eight / twelve chunks: the second of
        // those calls, mean of eight draws of requests, 131 / 123 / 121 / 121; its rows in any order, all with adapters, 134 / 137 / 139 / 141).
        p.chunks = (int)std::max<int64_t>(1, std::min<int64_t>((a.out + 31) / 32 / (3 * WARPS + 4), 6 * sm_count / (windows + rows / 64)));
        p.window_tiles = (int)std::min<int64_t>(most, std::max<int64_t>(WINDOW / 64 + 2, 4 * sm_count / (windows * p.chunks)));
        if (windows * p.window_tiles * p.chunks > 0x7fffffff) return 3;
        rc = launch_dependent(out ? low_rank_up_kernel<T, D, RB, true> : low_rank_up_kernel<T, D, RB, false>, p,
                (unsigned)(windows * p.window_tiles * p.chunks), THREADS, sizeof(UpShared<T, D, RB>), st);
        if (rc != 0) return rc;
        count_launch();
    }
    return 0;
}

template <typename T, typename D, int RB> int launch_rank(LowRankPlan &p, int sm_count, cudaStream_t st) {
    const LowRankArgs &a = p.a;
    auto aligned = [](const void *ptr, int64_t bytes, int64_t stride0, int64_t stride1) {
        return (uintptr_t)ptr % bytes == 0 && stride0 * 2 % bytes == 0 && stride1 * 2 % bytes == 0;
    };
    p.down_mode = a.down_in == 1 && a.in % 8 == 0 && aligned(a.down, 16, a.down_adapter, a.down_rank) ? VECTOR_OUTER
            : a.down_rank == 1 && a.rank % (2 * RB) == 0 && aligned(a.down, std::min(4 * RB, 16), a.down_adapter, a.down_in) ? VECTOR_RANK
                                                                                                                          : ELEMENTS;
    p.up_mode = a.up_out == 1 && a.out % 4 == 0 && aligned(a.up, 8, a.up_adapter, a.up_rank) ? VECTOR_OUTER
            : a.up_rank == 1 && a.rank % (4 * RB) == 0 && aligned(a.up, std::min(8 * RB, 16), a.up_adapter, a.up_out) ? VECTOR_RANK
                                                                                                                   : ELEMENTS;
    // whether each side is read and written in wide accesses
    const bool in = a.in % 8 == 0 && rows_aligned(a.src, a.src_ld * 2, a.rows) && p.down_mode != ELEMENTS;
    const bool out = a.out % 8 == 0 && rows_aligned(a.dst, a.dst_ld * (int)sizeof(D), a.rows)
            && (!a.base || rows_aligned(a.base, a.base_ld * (int)sizeof(D), a.rows)) && p.up_mode != ELEMENTS;
    if (!p.middle) return in && out ? launch_few<T, D, RB, true>(p, sm_count, st) : launch_few<T, D, RB, false>(p, sm_count, st);
    return launch_many<T, D, RB>(p, in, out, sm_count, st);
}

template <typename T, typename D> int launch_typed(LowRankPlan &p, int sm_count, cudaStream_t st) {
    if (p.a.rank <= 16) return launch_rank<T, D, 1>(p, sm_count, st);
    if (p.a.rank <= 32) return launch_rank<T, D, 2>(p, sm_count, st);
    if (p.a.rank <= 64) return launch_rank<T, D, 4>(p, sm_count, st);
    return launch_rank<T, D, 8>(p, sm_count, st);
}

} // namespace

// What one launch serves: above, tiles of 16 rows read the weights too often (us a call, one launch / two: 64 adapters 4096 x 4096, rank
// 16, 100 rows 9.1 / 9.9, 400 10.6 / 15.9, 1024 20.9 / 29.0, 2048 38.2 / 43.5; 16 adapters 4096 x 11008, rank 32, 512 rows 20.9 / 26.9,
// 1024 36.4 / 36.7, 2048 55.3 / 45.6; rank 64, 64 adapters 4096 x 4096, 400 rows 33.9 / 36.8, 1024 62.2 / 46.4).  What decides is how many
// rows share an adapter and how large its factors are, which is not known before the call (the indices are in device memory): the
// limit is where the two are even for 16 adapters, and for 64 some 14 % are lost at 2048 rows.  (The cluster of four CTAs was
// compared with two and eight on the 61 rows above only.)
static bool few_rows(int64_t rows, int64_t rank) { return rows <= (rank <= 32 ? 1024 : 512); }

size_t low_rank_scratch_bytes(int64_t rows, int64_t rank) {
    if (rows >= 0 && few_rows(rows, rank < 0 ? LOW_RANK_MAX : rank)) return 0;
    const int64_t blocks = rank < 0 || rank > 64 ? 8 : rank > 32 ? 4 : rank > 16 ? 2 : 1;
    return (size_t)(rows < 0 ? LOW_RANK_CHUNK : std::min<int64_t>(rows, LOW_RANK_CHUNK)) * 16 * blocks * sizeof(float) * LOW_RANK_SPLITS;
}

int launch_low_rank(const LowRankArgs &a, void *scratch, int sm_count, cudaStream_t st) {
    if (a.rows == 0 || a.out == 0) return 0;
    LowRankPlan p {};
    p.a = a;
    p.middle = few_rows(a.rows, a.rank) ? nullptr : (float *)scratch;
    if (a.dt == DT_BF16)
        return a.dst_dt == DT_F32 ? launch_typed<__nv_bfloat16, float>(p, sm_count, st) : launch_typed<__nv_bfloat16, __nv_bfloat16>(p, sm_count, st);
    if (a.dt == DT_F16) return a.dst_dt == DT_F32 ? launch_typed<__half, float>(p, sm_count, st) : launch_typed<__half, __half>(p, sm_count, st);
    return 3;
}

} // namespace qmm

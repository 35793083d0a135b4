// Low-rank adapters of many requests beside a shared projection, in one launch:
//   dst_t = base_t + scale_i (x_t down_i) up_i,  i = indices[t]; a row whose index names no adapter is base_t
// Bound by memory: of a row its src, base and dst cross it once, of an adapter its weights for each tile (from L2 but the first
// time); with ranks up to 128 there are 2 to 60 operations a byte, which mma.sync keeps up with.
//
// Rows are looked at in windows of 512.  The rows of a window that share an adapter make tiles of up to 16 MT rows, wherever
// they stand; a cluster of CTAs takes a tile: each CTA multiplies its share of the src's columns with the first factor, the
// sums of [rows][rank] meet in the CTAs' shared memory, and each CTA multiplies them with its share of the second factor's columns.
// So the products' middle never leaves the chip, and a single row's weights are streamed by a whole cluster.
// Operands go from global memory to the registers of an MMA without shared memory: a lane reads 16 bytes, and which eight of
// the summed (or of the output's) columns these are is decided alike for both operands, so any order serves.
// The middle is a 32-bit sum.  The second product takes it as a sum of 16-bit parts, most significant first: two (what is left
// out is 2^-18 of a value), or three where dst has 32 bits and the parts are bf16 (2^-27).  f16 parts are made of values that a
// power of two brings just below the type's largest, row by row.
#include <algorithm>

#include "launch.h"
#include "token_rows.cuh"

namespace qmm {

namespace {

constexpr int THREADS = 256, WARPS = THREADS / 32, WINDOW = 512;

enum : int { VECTOR_OUTER = 0, VECTOR_RANK = 1, ELEMENTS = 2 }; // which neighbours of a factor a lane reads at once

struct LowRankPlan {
    LowRankArgs a;
    int cluster; // CTAs of a tile
    int window_clusters; // clusters that take a window's tiles in turn
    int down_mode, up_mode;
};

template <int RB> constexpr int M_TILES = RB <= 2 ? 4 : RB == 4 ? 2 : 1; // of 16 rows each
template <int RB> struct Layout { // of shared memory
    static constexpr int ROWS = 16 * M_TILES<RB>, RANK = 16 * RB, PITCH = RANK + 4;
    float slabs[WARPS / 2][ROWS][PITCH]; // sums of pairs of warps; later the second product's operand
    alignas(16) float part[ROWS][RANK]; // this CTA's sums, which the whole cluster reads
    float unit[ROWS]; // f16: the power of two that a row's sums were divided by
    alignas(16) int index[WINDOW];
    unsigned short place[WINDOW]; // rows before it in the window with the same index
    unsigned short first[WINDOW]; // first row of each tile
    unsigned short rows[ROWS]; // of the tile
    int counts[2 * WARPS];
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

// eight 16-bit values of a row from `col` on, zeros behind its end
template <bool VEC> __device__ __forceinline__ uint4 load_8(const uint16_t *row, int64_t col, int64_t cols) {
    if constexpr (VEC) {
        return col < cols ? ptx::ld_dependent((const uint4 *)(row + col)) : make_uint4(0, 0, 0, 0);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t lo = col + 2 * i < cols ? ld_u16(row + col + 2 * i) : 0u;
            const uint32_t hi = col + 2 * i + 1 < cols ? ld_u16(row + col + 2 * i + 1) : 0u;
            w[i] = lo | hi << 16;
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// The first factor's operand of 32 columns of src, of which this lane has eight from k on: w[j] = (pairs of) those of column
// n(j0 + j, lane / 4) of the rank, where n(j, g) is 8 j + g, or 2 RB g + j where neighbours are read along the rank.
template <int RB, int J, bool VEC>
__device__ __forceinline__ void load_down(uint32_t (&w)[J][4], const LowRankPlan &p, const uint16_t *down, int64_t k, int j0, int lane) {
    const LowRankArgs &a = p.a;
    const int g = lane >> 2;
    if (p.down_mode == VECTOR_OUTER) {
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int n = 8 * (j0 + j) + g;
            const uint4 v = n < a.rank && k < a.in ? ptx::ld_dependent((const uint4 *)(down + n * a.down_rank + k)) : make_uint4(0, 0, 0, 0);
            w[j][0] = v.x; w[j][1] = v.y; w[j][2] = v.z; w[j][3] = v.w;
        }
    } else if (VEC || p.down_mode == VECTOR_RANK) {
        uint32_t rows[8][J / 2]; // two columns of the rank a word
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const bool there = 2 * RB * g < a.rank && k + i < a.in;
            const uint16_t *at = down + (k + i) * a.down_in + 2 * RB * g + j0;
#pragma unroll
            for (int q = 0; q < J / 2; ++q) rows[i][q] = 0;
            if (there) {
                if constexpr (J == 2) rows[i][0] = ld_u32(at);
                else if constexpr (J == 4) {
                    const uint2 v = ptx::ld_dependent((const uint2 *)at);
                    rows[i][0] = v.x; rows[i][1] = v.y;
                } else {
                    const uint4 v = ptx::ld_dependent((const uint4 *)at);
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
            const int n = 8 * (j0 + j) + g;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint16_t *at = down + n * a.down_rank + (k + 2 * i) * a.down_in;
                const uint32_t lo = n < a.rank && k + 2 * i < a.in ? ld_u16(at) : 0u;
                const uint32_t hi = n < a.rank && k + 2 * i + 1 < a.in ? ld_u16(at + a.down_in) : 0u;
                w[j][i] = lo | hi << 16;
            }
        }
    }
}

// column of the rank that value i (of four) of a lane is, in the second product's step s
template <int RB> __device__ __forceinline__ int rank_column(int mode, int s, int t, int i) {
    return mode == VECTOR_RANK ? t * 4 * RB + 4 * s + i : 16 * s + 4 * t + i;
}

// The second factor's operand of 32 columns of dst from n0 on: w[j] = this lane's values of the rank at column n0 + 8 (g / 2) + 2 j + g % 2.
template <int RB, bool VEC>
__device__ __forceinline__ void load_up(uint32_t (&w)[4][RB][2], const LowRankPlan &p, const uint16_t *up, int64_t n0, int lane) {
    const LowRankArgs &a = p.a;
    const int g = lane >> 2, t = lane & 3;
    const int64_t n = n0 + 8 * (g >> 1);
    if (p.up_mode == VECTOR_OUTER) {
#pragma unroll
        for (int s = 0; s < RB; ++s) {
            uint4 rows[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int k = 16 * s + 4 * t + i;
                rows[i] = k < a.rank && n < a.out ? ptx::ld_dependent((const uint4 *)(up + k * a.up_rank + n)) : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                w[0][s][h] = halves(rows[2 * h].x, rows[2 * h + 1].x, g & 1);
                w[1][s][h] = halves(rows[2 * h].y, rows[2 * h + 1].y, g & 1);
                w[2][s][h] = halves(rows[2 * h].z, rows[2 * h + 1].z, g & 1);
                w[3][s][h] = halves(rows[2 * h].w, rows[2 * h + 1].w, g & 1);
            }
        }
    } else if (VEC || p.up_mode == VECTOR_RANK) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t col = n + 2 * j + (g & 1);
            const bool there = col < a.out && t * 4 * RB < a.rank;
            const uint16_t *at = up + col * a.up_out + t * 4 * RB;
            if constexpr (RB == 1) {
                const uint2 v = there ? ptx::ld_dependent((const uint2 *)at) : make_uint2(0, 0);
                w[j][0][0] = v.x; w[j][0][1] = v.y;
            } else {
#pragma unroll
                for (int s = 0; s < RB; s += 2) {
                    const uint4 v = there ? ptx::ld_dependent((const uint4 *)(at + 4 * s)) : make_uint4(0, 0, 0, 0);
                    w[j][s][0] = v.x; w[j][s][1] = v.y; w[j][s + 1][0] = v.z; w[j][s + 1][1] = v.w;
                }
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t col = n + 2 * j + (g & 1);
#pragma unroll
            for (int s = 0; s < RB; ++s)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int k = 16 * s + 4 * t + 2 * h;
                    const uint16_t *at = up + col * a.up_out + k * a.up_rank;
                    const uint32_t lo = col < a.out && k < a.rank ? ld_u16(at) : 0u;
                    const uint32_t hi = col < a.out && k + 1 < a.rank ? ld_u16(at + a.up_rank) : 0u;
                    w[j][s][h] = lo | hi << 16;
                }
        }
    }
}

// eight values of base or dst
template <typename D, bool VEC> struct Eight {
    uint4 raw[sizeof(D) / 2];
    __device__ __forceinline__ void load(const D *row, int64_t col, int64_t cols) {
        if constexpr (sizeof(D) == 2) {
            raw[0] = load_8<VEC>((const uint16_t *)row, col, cols);
        } else if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < 2; ++i) raw[i] = col < cols ? ptx::ld_dependent((const uint4 *)(row + col) + i) : make_uint4(0, 0, 0, 0);
        } else {
            uint32_t w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = col + i < cols ? ld_u32(row + col + i) : 0u;
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
    static __device__ __forceinline__ void store(D *row, int64_t col, int64_t cols, const float (&v)[8]) {
        if constexpr (VEC) {
            Cols<D, true>::store(row, col, cols, v);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (col + i < cols) row[col + i] = from_f32<D>(v[i]);
        }
    }
};

// The sums of this warp's share of the src's columns, U steps of 32 at a time, for the first M of the tile's groups of 16 rows.
template <typename T, int RB, bool VEC, int M, int U, int MT>
__device__ __forceinline__ void first_product(float (&acc)[MT][2 * RB][4], const LowRankPlan &p, const uint16_t *down, const Layout<RB> &sh,
        int64_t window, int count, int lane, int64_t first, int64_t step) {
    const LowRankArgs &a = p.a;
    constexpr int J = 2 * RB < 8 ? 2 * RB : 8; // blocks of eight of the rank at a time
    uint32_t pair[M]; // rows g and g + 8
#pragma unroll
    for (int m = 0; m < M; ++m)
        pair[m] = sh.rows[min(16 * m + (lane >> 2), count - 1)] | (uint32_t)sh.rows[min(16 * m + 8 + (lane >> 2), count - 1)] << 16;
    const uint16_t *src = (const uint16_t *)a.src + window * a.src_ld;
    const int64_t steps = (a.in + 31) / 32;
    for (int64_t s = first; s < steps; s += U * step) {
        uint4 x[U][M][2];
        uint32_t w[U][J][4];
#pragma unroll
        for (int u = 0; u < U; ++u) { // (steps behind the last read zeros)
            const int64_t k = (s + u * step) * 32 + 8 * (lane & 3);
#pragma unroll
            for (int m = 0; m < M; ++m) {
                x[u][m][0] = load_8<VEC>(src + (pair[m] & 0xffff) * a.src_ld, k, a.in);
                x[u][m][1] = load_8<VEC>(src + (pair[m] >> 16) * a.src_ld, k, a.in);
            }
            load_down<RB, J, VEC>(w[u], p, down, k, 0, lane);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j0 = 0; j0 < 2 * RB; j0 += J) {
                if (j0 > 0) load_down<RB, J, VEC>(w[u], p, down, (s + u * step) * 32 + 8 * (lane & 3), j0, lane);
#pragma unroll
                for (int m = 0; m < M; ++m)
#pragma unroll
                    for (int j = 0; j < J; ++j) {
                        mma_16816<T>(acc[m][j0 + j], x[u][m][0].x, x[u][m][1].x, x[u][m][0].y, x[u][m][1].y, w[u][j][0], w[u][j][1]);
                        mma_16816<T>(acc[m][j0 + j], x[u][m][0].z, x[u][m][1].z, x[u][m][0].w, x[u][m][1].w, w[u][j][2], w[u][j][3]);
                    }
            }
    }
}

template <typename T, typename D, int RB, bool VEC>
__global__ void __launch_bounds__(THREADS, VEC ? 2 : 1) low_rank_kernel(const __grid_constant__ LowRankPlan p) {
    extern __shared__ __align__(16) unsigned char shared[];
    Layout<RB> &sh = *reinterpret_cast<Layout<RB> *>(shared);
    constexpr int MT = M_TILES<RB>, TM = 16 * MT;
    constexpr int PARTS = sizeof(D) == 4 && std::is_same<T, __nv_bfloat16>::value ? 3 : 2;
    static_assert(sizeof(uint4) * PARTS * MT * RB * 32 <= sizeof(sh.slabs), "the operand lies where the slabs were");
    ptx::grid_dependency_wait();
    const LowRankArgs &a = p.a;
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32, rank = (int)cluster_rank();
    const int number = (int)blockIdx.x / p.cluster; // of the cluster
    const int64_t window = (int64_t)(number / p.window_clusters) * WINDOW;
    const int rows = (int)min((int64_t)WINDOW, a.rows - window);

    // the window's tiles: a row that has a multiple of TM rows of its index before it is the first of one
    for (int i = threadIdx.x; i < WINDOW; i += THREADS) {
        int id = -1; // behind the last row
        if (i < rows) {
            id = ptx::ld_dependent(a.indices + window + i);
            if ((unsigned)id >= (unsigned)a.adapters) id = a.adapters;
        }
        sh.index[i] = id;
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int i = h * THREADS + threadIdx.x, id = sh.index[i], whole = (i & ~31) / 4;
        int before = 0;
        for (int q = 0; q < whole; ++q) { // all rows before this warp's
            const int4 v = *reinterpret_cast<const int4 *>(sh.index + 4 * q);
            before += (v.x == id) + (v.y == id) + (v.z == id) + (v.w == id);
        }
        before += __popc(__match_any_sync(0xffffffffu, id) & ((1u << lane) - 1));
        sh.place[i] = (unsigned short)before;
        const uint32_t firsts = __ballot_sync(0xffffffffu, id >= 0 && before % TM == 0);
        if (lane == 0) sh.counts[h * WARPS + warp] = __popc(firsts);
    }
    __syncthreads();
    int tiles = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int i = h * THREADS + threadIdx.x;
        int at = 0;
        tiles = 0;
        for (int q = 0; q < 2 * WARPS; ++q) {
            if (q == h * WARPS + warp) at = tiles;
            tiles += sh.counts[q];
        }
        const bool leads = sh.index[i] >= 0 && sh.place[i] % TM == 0;
        const uint32_t firsts = __ballot_sync(0xffffffffu, leads);
        if (leads) sh.first[at + __popc(firsts & ((1u << lane) - 1))] = (unsigned short)i;
    }

    bool arrived = false; // at the barrier behind the reads of `part`
    for (int tile = number % p.window_clusters; tile < tiles; tile += p.window_clusters) {
        __syncthreads();
        const int lead = sh.first[tile], id = sh.index[lead], base_place = sh.place[lead];
        int count = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int i = h * THREADS + threadIdx.x, at = sh.place[i] - base_place;
            const bool mine = sh.index[i] == id && at >= 0 && at < TM;
            if (mine) sh.rows[at] = (unsigned short)i;
            count += __syncthreads_count(mine);
        }
        const int64_t blocks = (a.out + 31) / 32; // of 32 columns of dst, in runs of neighbours for each CTA
        const int64_t first_block = blocks * rank / p.cluster + warp, end_block = blocks * (rank + 1) / p.cluster;
        if (id == a.adapters) { // no adapter
            if (a.base == a.dst && a.base_ld == a.dst_ld) continue; // in place
            for (int64_t b = first_block; b < end_block; b += WARPS) {
                const int64_t col = 32 * b + 8 * (lane & 3);
                for (int r = lane >> 2; r < count; r += 8) {
                    const int64_t row = window + sh.rows[r];
                    float v[8] = {};
                    if (a.base) {
                        Eight<D, VEC> e;
                        e.load((const D *)a.base + row * a.base_ld, col, a.out);
                        e.get(v);
                    }
                    Eight<D, VEC>::store((D *)a.dst + row * a.dst_ld, col, a.out, v);
                }
            }
            continue;
        }
        const uint16_t *down = (const uint16_t *)a.down + id * a.down_adapter, *up = (const uint16_t *)a.up + id * a.up_adapter;
        const int groups = (count + 15) / 16;

        float acc[MT][2 * RB][4];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int j = 0; j < 2 * RB; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[m][j][i] = 0.f;
        const int64_t first = (int64_t)rank * WARPS + warp, step = (int64_t)p.cluster * WARPS;
        if (groups == 1) first_product<T, RB, VEC, 1, (!VEC || RB > 2) ? 1 : 4 / RB>(acc, p, down, sh, window, count, lane, first, step);
        else first_product<T, RB, VEC, MT, 1>(acc, p, down, sh, window, count, lane, first, step);

        // the warps' sums: the upper four warps', then with them the lower four's
        auto column = [&](int j, int c) { return p.down_mode == VECTOR_RANK ? 2 * RB * c + j : 8 * j + c; };
#pragma unroll
        for (int round = 0; round < 2; ++round) {
            if ((warp < WARPS / 2) == (round == 1)) {
#pragma unroll
                for (int m = 0; m < MT; ++m)
                    if (m < groups)
#pragma unroll
                        for (int j = 0; j < 2 * RB; ++j)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                float *at = &sh.slabs[warp % (WARPS / 2)][16 * m + 8 * (i / 2) + (lane >> 2)][column(j, 2 * (lane & 3) + i % 2)];
                                *at = round ? acc[m][j][i] + *at : acc[m][j][i];
                            }
            }
            __syncthreads();
        }
        if (arrived) cluster_wait(); // (the last tile's `part` has been read everywhere)
        for (int i = threadIdx.x; i < groups * 16 * 16 * RB; i += THREADS) {
            const int row = i / (16 * RB), col = i % (16 * RB);
            sh.part[row][col] = (sh.slabs[0][row][col] + sh.slabs[1][row][col]) + (sh.slabs[2][row][col] + sh.slabs[3][row][col]);
        }
        cluster_arrive();
        cluster_wait();

        // The second product's operand: a thread has the values of a row that one lane of an MMA needs.
        uint4 *operand = reinterpret_cast<uint4 *>(sh.slabs);
        {
            const int row = threadIdx.x / 4, t = threadIdx.x % 4;
            float v[RB][4];
            float most = 0.f;
            if (row < groups * 16) {
                const float scale = a.scales ? ptx::ld_dependent(a.scales + id) : 1.f;
                const uint32_t part = ptx::smem_u32(sh.part[row]);
#pragma unroll
                for (int s = 0; s < RB; ++s) {
                    const int col = rank_column<RB>(p.up_mode, s, t, 0);
                    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
                    for (int c = 0; c < p.cluster; ++c) {
                        const float4 q = ld_cluster(peer_address(part + 4 * col, c));
                        sum.x += q.x; sum.y += q.y; sum.z += q.z; sum.w += q.w;
                    }
                    v[s][0] = sum.x; v[s][1] = sum.y; v[s][2] = sum.z; v[s][3] = sum.w;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        v[s][i] = col + i < a.rank ? v[s][i] * scale : 0.f; // (zeros whatever src holds)
                        most = fmaxf(most, fabsf(v[s][i]));
                    }
                }
            }
            float unit = 1.f;
            if constexpr (std::is_same<T, __half>::value) { // the largest of the row into [2^13, 2^14)
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
                if (most > 0.f && most < INFINITY) unit = __uint_as_float(max((__float_as_uint(most) & 0x7f800000u), 87u << 23)) * 0x1p-13f;
                if (t == 0 && row < TM) sh.unit[row] = unit;
            }
            if (row < groups * 16) {
                const float inverse = 1.f / unit; // (a power of two)
                const int at = (row / 16 * RB) * 32 + row % 8 * 4 + t, word = row % 16 / 8;
#pragma unroll
                for (int s = 0; s < RB; ++s) {
                    float rest[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) rest[i] = v[s][i] * inverse;
#pragma unroll
                    for (int q = 0; q < PARTS; ++q) {
                        uint32_t *to = reinterpret_cast<uint32_t *>(operand + (q * MT * RB + s) * 32 + at) + word;
                        T part[4];
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
            }
        }
        cluster_arrive();
        arrived = true;
        __syncthreads();

        for (int64_t b = first_block; b < end_block; b += WARPS) {
            const int64_t n0 = 32 * b, col = n0 + 8 * (lane & 3);
            uint32_t w[4][RB][2];
            constexpr int AHEAD = MT == 1 ? 1 : sizeof(D) == 4 ? 2 : MT; // groups of 16 rows whose base is read together
            Eight<D, VEC> base[AHEAD][2];
#pragma unroll
            for (int m0 = 0; m0 < MT; m0 += AHEAD) {
                if (m0 >= groups) break;
                if (a.base) {
#pragma unroll
                    for (int m = 0; m < AHEAD; ++m)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int r = min(16 * (m0 + m) + 8 * h + (lane >> 2), count - 1);
                            if (m0 + m < groups) base[m][h].load((const D *)a.base + (window + sh.rows[r]) * a.base_ld, col, a.out);
                        }
                }
                if (m0 == 0) load_up<RB, VEC>(w, p, up, n0, lane);
#pragma unroll
                for (int m = 0; m < AHEAD; ++m) {
                    if (m0 + m >= groups) break;
                    float out[4][4];
                    float unit[2] = {1.f, 1.f};
                    if constexpr (std::is_same<T, __half>::value) {
                        unit[0] = sh.unit[16 * (m0 + m) + (lane >> 2)];
                        unit[1] = sh.unit[16 * (m0 + m) + (lane >> 2) + 8];
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float v[8] = {};
                        if (a.base) base[m][h].get(v);
                        const float inverse = 1.f / unit[h];
#pragma unroll
                        for (int j = 0; j < 4; ++j)
#pragma unroll
                            for (int i = 0; i < 2; ++i)
                                out[j][2 * h + i] = std::is_same<T, __half>::value ? v[2 * j + i] * inverse : v[2 * j + i];
                    }
#pragma unroll
                    for (int q = PARTS - 1; q >= 0; --q) // the smallest first
#pragma unroll
                        for (int s = 0; s < RB; ++s) {
                            const uint4 f = operand[((q * MT + m0 + m) * RB + s) * 32 + lane];
#pragma unroll
                            for (int j = 0; j < 4; ++j) mma_16816<T>(out[j], f.x, f.y, f.z, f.w, w[j][s][0], w[j][s][1]);
                        }
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int r = 16 * (m0 + m) + 8 * h + (lane >> 2);
                        float v[8];
#pragma unroll
                        for (int j = 0; j < 4; ++j)
#pragma unroll
                            for (int i = 0; i < 2; ++i)
                                v[2 * j + i] = std::is_same<T, __half>::value ? out[j][2 * h + i] * unit[h] : out[j][2 * h + i];
                        if (r < count) Eight<D, VEC>::store((D *)a.dst + (window + sh.rows[r]) * a.dst_ld, col, a.out, v);
                    }
                }
            }
        }
    }
    if (arrived) cluster_wait(); // nobody leaves while its sums may be read
}

template <typename T, typename D, int RB, bool VEC> int launch_kernel(const LowRankPlan &p, cudaStream_t st) {
    static std::atomic<unsigned long long> done;
    if (!opt_in_dynamic_smem(low_rank_kernel<T, D, RB, VEC>, (int)sizeof(Layout<RB>), done)) return 5;
    const int64_t windows = (p.a.rows + WINDOW - 1) / WINDOW;
    cudaLaunchConfig_t cfg {};
    cfg.gridDim = dim3((unsigned)(windows * p.window_clusters * p.cluster));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = sizeof(Layout<RB>);
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
    return cudaLaunchKernelExC(&cfg, (const void *)low_rank_kernel<T, D, RB, VEC>, kargs) == cudaSuccess ? 0 : 5;
}

template <typename T, typename D, int RB> int launch_rank(LowRankPlan &p, int sm_count, cudaStream_t st) {
    const LowRankArgs &a = p.a;
    constexpr int TM = 16 * M_TILES<RB>;
    bool vec = a.in % 8 == 0 && a.out % 8 == 0 && rows_aligned(a.src, a.src_ld * 2, a.rows)
            && rows_aligned(a.dst, a.dst_ld * (int)sizeof(D), a.rows) && (!a.base || rows_aligned(a.base, a.base_ld * (int)sizeof(D), a.rows));
    auto aligned = [](const void *ptr, int64_t bytes, int64_t stride0, int64_t stride1) {
        return (uintptr_t)ptr % bytes == 0 && stride0 * 2 % bytes == 0 && stride1 * 2 % bytes == 0;
    };
    p.down_mode = a.down_in == 1 && a.in % 8 == 0 && aligned(a.down, 16, a.down_adapter, a.down_rank) ? VECTOR_OUTER
            : a.down_rank == 1 && a.rank % (2 * RB) == 0 && aligned(a.down, std::min(4 * RB, 16), a.down_adapter, a.down_in) ? VECTOR_RANK
                                                                                                                          : ELEMENTS;
    p.up_mode = a.up_out == 1 && a.out % 8 == 0 && aligned(a.up, 16, a.up_adapter, a.up_rank) ? VECTOR_OUTER
            : a.up_rank == 1 && a.rank % (4 * RB) == 0 && aligned(a.up, std::min(8 * RB, 16), a.up_adapter, a.up_out) ? VECTOR_RANK
                                                                                                                   : ELEMENTS;
    vec = vec && p.down_mode != ELEMENTS && p.up_mode != ELEMENTS;
    const int64_t windows = (a.rows + WINDOW - 1) / WINDOW, rows = std::min<int64_t>(a.rows, WINDOW);
    p.cluster = a.rows <= 64 ? 8 : 4;
    p.window_clusters = (int)std::min<int64_t>(rows, std::max<int64_t>(WINDOW / TM + 2, 2 * sm_count / (windows * p.cluster)));
    if (windows * p.window_clusters * p.cluster > 0x7fffffff) return 3;
    const int rc = vec ? launch_kernel<T, D, RB, true>(p, st) : launch_kernel<T, D, RB, false>(p, st);
    if (rc == 0) count_launch();
    return rc;
}

template <typename T, typename D> int launch_typed(LowRankPlan &p, int sm_count, cudaStream_t st) {
    if (p.a.rank <= 16) return launch_rank<T, D, 1>(p, sm_count, st);
    if (p.a.rank <= 32) return launch_rank<T, D, 2>(p, sm_count, st);
    if (p.a.rank <= 64) return launch_rank<T, D, 4>(p, sm_count, st);
    return launch_rank<T, D, 8>(p, sm_count, st);
}

} // namespace

int launch_low_rank(const LowRankArgs &a, int sm_count, cudaStream_t st) {
    if (a.rows == 0 || a.out == 0) return 0;
    LowRankPlan p {};
    p.a = a;
    if (a.dt == DT_BF16)
        return a.dst_dt == DT_F32 ? launch_typed<__nv_bfloat16, float>(p, sm_count, st) : launch_typed<__nv_bfloat16, __nv_bfloat16>(p, sm_count, st);
    if (a.dt == DT_F16) return a.dst_dt == DT_F32 ? launch_typed<__half, float>(p, sm_count, st) : launch_typed<__half, __half>(p, sm_count, st);
    return 3;
}

} // namespace qmm

// What the kernels that move and sum rows of tokens share: a thread's share of a row's columns, in two forms, and the
// random words of dropout.
//
// VEC: eight neighbouring columns, 16-byte accesses; every row of every tensor starts on a 16-byte boundary and holds a
// multiple of eight columns.  Otherwise: four columns, 32 apart, so that a warp covers
// 128 neighbouring ones and its accesses stay contiguous wherever the rows start; with dropout the 128 begin at a
// multiple of four elements of the whole tensor, up to three columns before the row.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "sm100_ptx.cuh"
#include "token_ops.h"

namespace qmm {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

__device__ __forceinline__ void unpack2(uint32_t u, float &lo, float &hi, __nv_bfloat16) {
    lo = __uint_as_float(u << 16);
    hi = __uint_as_float(u & 0xffff0000u);
}
__device__ __forceinline__ void unpack2(uint32_t u, float &lo, float &hi, __half) {
    const float2 f = __half22float2(*reinterpret_cast<__half2 *>(&u));
    lo = f.x;
    hi = f.y;
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __nv_bfloat16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __half) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
}

template <typename T, bool VEC> struct Cols;

template <typename T> struct Cols<T, true> {
    static constexpr int N = 8;
    uint4 raw[sizeof(T) / 2];
    // of a row with a multiple of eight columns (one predicate and no branch: rows' loads stay together); zeros beyond it
    __device__ __forceinline__ void load(const T *row, int64_t col, int64_t cols) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
            raw[i] = make_uint4(0, 0, 0, 0);
            if (col < cols) raw[i] = ptx::ld_dependent((const uint4 *)(row + col) + i);
        }
    }
    // of the `left` columns that a row still has from p on
    __device__ __forceinline__ void load_ragged(const T *p, int64_t left) {
        if (left >= 8) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i) raw[i] = ptx::ld_dependent((const uint4 *)p + i);
        } else {
            T part[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) part[i] = i < left ? p[i] : from_f32<T>(0.f);
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i) raw[i] = reinterpret_cast<const uint4 *>(part)[i];
        }
    }
    __device__ __forceinline__ void load_shared(const T *p) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) raw[i] = reinterpret_cast<const uint4 *>(p)[i];
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                v[4 * i] = __uint_as_float(raw[i].x);
                v[4 * i + 1] = __uint_as_float(raw[i].y);
                v[4 * i + 2] = __uint_as_float(raw[i].z);
                v[4 * i + 3] = __uint_as_float(raw[i].w);
            }
        } else {
            unpack2(raw[0].x, v[0], v[1], T());
            unpack2(raw[0].y, v[2], v[3], T());
            unpack2(raw[0].z, v[4], v[5], T());
            unpack2(raw[0].w, v[6], v[7], T());
        }
    }
    static __device__ __forceinline__ void store(T *row, int64_t col, int64_t cols, const float (&v)[8]) {
        if (col < cols) store_ragged(row + col, 8, v);
    }
    static __device__ __forceinline__ void store_ragged(T *p, int64_t left, const float (&v)[8]) {
        if (left >= 8) {
            if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    reinterpret_cast<float4 *>(p)[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
            } else {
                *reinterpret_cast<uint4 *>(p) = make_uint4(pack2(v[0], v[1], T()), pack2(v[2], v[3], T()),
                        pack2(v[4], v[5], T()), pack2(v[6], v[7], T()));
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < left) p[i] = from_f32<T>(v[i]);
        }
    }
};

template <typename T> struct Cols<T, false> {
    static constexpr int N = 4;
    T raw[4];
    // of 32 i: the columns that are there (those below 0 are among the first 32)
    static __device__ __forceinline__ bool there(int i, int64_t col, int64_t cols) {
        return (i > 0 || col >= 0) && 32 * i < (int)min((int64_t)128, cols - col);
    }
    __device__ __forceinline__ void load(const T *row, int64_t col, int64_t cols) {
        const T *p = row + col;
#pragma unroll
        for (int i = 0; i < 4; ++i) raw[i] = there(i, col, cols) ? p[32 * i] : from_f32<T>(0.f);
    }
    __device__ __forceinline__ void get(float (&v)[4]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = to_f32(raw[i]);
    }
    static __device__ __forceinline__ void store(T *row, int64_t col, int64_t cols, const float (&v)[4]) {
        T *p = row + col;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (there(i, col, cols)) p[32 * i] = from_f32<T>(v[i]);
    }
};

// Shares of a row: `units` threads cover it (a multiple of 32 where a warp works together).
template <bool VEC> __host__ __device__ inline int64_t row_units(int64_t cols, bool dropout) {
    return VEC ? (cols + 7) / 8 : (cols + (dropout ? 3 : 0) + 127) / 128 * 32;
}

// First column of share `unit` of row t.
template <bool VEC> __device__ __forceinline__ int64_t unit_column(int64_t unit, int64_t t, int64_t cols, bool dropout) {
    if (VEC) return unit * 8;
    return (unit >> 5) * 128 + (unit & 31) - (dropout ? (t * cols) & 3 : 0);
}

// Philox4x32 with ten rounds (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3; 2011): the four
// words of block `block` under key `seed`; the upper half of the counter is the caller's offset.
__device__ __forceinline__ uint4 philox(uint64_t seed, uint64_t offset, uint64_t block) {
    uint32_t x0 = (uint32_t)block, x1 = (uint32_t)(block >> 32), x2 = (uint32_t)offset, x3 = (uint32_t)(offset >> 32);
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t a = (uint64_t)x0 * 0xD2511F53u, b = (uint64_t)x2 * 0xCD9E8D57u;
        x0 = (uint32_t)(b >> 32) ^ x1 ^ k0;
        x2 = (uint32_t)(a >> 32) ^ x3 ^ k1;
        x1 = (uint32_t)b;
        x3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return make_uint4(x0, x1, x2, x3);
}

// A value that is the same in every lane of a warp, told to the compiler: the result of a reduction over the warp lives in a
// uniform register.  (The ten rounds' keys are then made beside the lanes' own work: 8.4 M blocks 33.0 -> 26.9 us.)
__device__ __forceinline__ uint64_t same_in_warp(uint64_t v) {
    const uint32_t lo = __reduce_or_sync(0xffffffffu, (uint32_t)v), hi = __reduce_or_sync(0xffffffffu, (uint32_t)(v >> 32));
    return (uint64_t)hi << 32 | lo;
}

// v[i] = kept ? v[i] * scale : 0 for a thread's share of row t.  Element i of the tensor (in row-major order of its
// logical dims) uses word i % 4 of block i / 4.  A dropped element is zero whatever it was, infinities and NaN included.
// `words`: 128 words of shared memory of this warp's own (unused by VEC); the whole warp calls it.
template <bool VEC, int N>
__device__ __forceinline__ void random_words(uint32_t (&u)[N], uint64_t seed, uint64_t offset, int64_t t, int64_t cols, int64_t col,
        uint32_t *words) {
    if constexpr (VEC) {
        const uint64_t block = (uint64_t)(t * cols + col) >> 2;
        const uint4 a = philox(seed, offset, block), b = philox(seed, offset, block + 1);
        u[0] = a.x; u[1] = a.y; u[2] = a.z; u[3] = a.w;
        u[4] = b.x; u[5] = b.y; u[6] = b.z; u[7] = b.w;
    } else {
        const int lane = threadIdx.x & 31;
        const uint64_t block = (uint64_t)(t * cols + col - lane) >> 2; // of the warp's first column
        __syncwarp();
        reinterpret_cast<uint4 *>(words)[lane] = philox(seed, offset, block + lane);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = words[32 * i + lane];
    }
}
template <int N> __device__ __forceinline__ void drop(float (&v)[N], const uint32_t (&u)[N], const DropoutState &d) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = u[i] >= d.threshold ? v[i] : 0.f;
}
template <bool VEC, int N>
__device__ __forceinline__ void apply_dropout(float (&v)[N], const DropoutState &d, uint64_t seed, uint64_t offset, int64_t t,
        int64_t cols, int64_t col, uint32_t *words) {
    if (d.drop_all) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = 0.f;
        return;
    }
    uint32_t u[N];
    random_words<VEC>(u, seed, offset, t, cols, col, words);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] *= d.scale;
    drop(v, u, d);
}

__device__ __forceinline__ uint64_t ld_dependent_u64(const int64_t *p) {
    uint64_t v;
    asm volatile("ld.global.u64 %0, [%1];" : "=l"(v) : "l"(p));
    return v;
}

// every row of the tensor starts on a 16-byte boundary
inline bool rows_aligned(const void *p, int64_t pitch_bytes, int64_t rows) {
    return (uintptr_t)p % 16 == 0 && (rows <= 1 || pitch_bytes % 16 == 0);
}

} // namespace qmm

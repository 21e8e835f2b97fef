// Shared device helpers for the gfx950 kernels of libterrace_hip.so.
#pragma once

#include <hip/hip_runtime.h>
#include <hip/hip_fp16.h>
#include <stdint.h>

#include "terrace_hip.h"

namespace terrace {

constexpr int kWave = 64;        // CDNA wavefront width
constexpr int kBlock = 256;      // default workgroup: 4 waves
constexpr int kWavesPerBlock = kBlock / kWave;

__device__ __forceinline__ int lane_id() { return threadIdx.x & (kWave - 1); }
__device__ __forceinline__ int wave_in_block() { return threadIdx.x >> 6; }

__device__ __forceinline__ uint64_t lanes_below(int lane) { return (1ull << lane) - 1ull; }

// Wave-private LDS words that lanes of one wave exchange values through.  The pointer carries the LDS address
// space in its type: a volatile access through a generic pointer is left as a flat instruction by the compiler,
// through one of these it is a ds_read / ds_write.
typedef __attribute__((address_space(3))) volatile int32_t lds_i32;
typedef __attribute__((address_space(3))) volatile float lds_f32;

// Value held by `src_lane` (uniform across the wave).
__device__ __forceinline__ int read_lane(int v, int src_lane) {
    return __builtin_amdgcn_readlane(v, src_lane);
}

// Butterfly exchange with lane ^ mask.  Distances 1 and 2 use DPP quad permutes, 4, 8 and 16 a
// ds_swizzle in bit mode (and-mask 0x1F, xor-mask the distance), 32 a ds_bpermute.
template <int MASK>
__device__ __forceinline__ int xchg_xor_i(int v) {
    if constexpr (MASK == 1) {
        return __builtin_amdgcn_update_dpp(v, v, 0xB1, 0xF, 0xF, false);   // quad_perm [1,0,3,2]
    } else if constexpr (MASK == 2) {
        return __builtin_amdgcn_update_dpp(v, v, 0x4E, 0xF, 0xF, false);   // quad_perm [2,3,0,1]
    } else if constexpr (MASK == 4) {
        return __builtin_amdgcn_ds_swizzle(v, 0x101F);                     // bit mode: xor 4
    } else if constexpr (MASK == 8) {
        return __builtin_amdgcn_ds_swizzle(v, 0x201F);                     // bit mode: xor 8
    } else if constexpr (MASK == 16) {
        return __builtin_amdgcn_ds_swizzle(v, 0x401F);                     // bit mode: xor 16
    } else {
        return __shfl_xor(v, 32, kWave);
    }
}
template <int MASK>
__device__ __forceinline__ float xchg_xor_f(float v) {
    return __int_as_float(xchg_xor_i<MASK>(__float_as_int(v)));
}

// Wave-wide inclusive/exclusive helpers over ints (used for small scans).
__device__ __forceinline__ int wave_inclusive_scan(int v) {
    const int lane = lane_id();
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
        int o = __shfl_up(v, d, kWave);
        if (lane >= d) v += o;
    }
    return v;
}

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

template <typename V>
__device__ __forceinline__ V ld_stream(const V *p) { return __builtin_nontemporal_load(p); }
template <typename V>
__device__ __forceinline__ void st_stream(V *p, V v) { __builtin_nontemporal_store(v, p); }

template <typename V>
__device__ __forceinline__ V zero_of() { return V(0); }
template <>
__device__ __forceinline__ u32x4 zero_of<u32x4>() { return u32x4{0u, 0u, 0u, 0u}; }

// Row ids a caller hands in are never trusted with an address: an id is used only if it lies in [0, bound),
// which one unsigned compare decides ((uint64_t)id < (uint64_t)bound is false for negative ids too).  An id
// outside is a dead entry -- a zero row for a gather, no contribution for the combine, a copy not made for a
// scatter.  The stage operators bound the planes their own index kernels wrote all the same.
__device__ __forceinline__ bool row_in(int64_t id, int64_t bound) { return (uint64_t)id < (uint64_t)bound; }

// Sum over the wave, in every lane: four rotations inside the rows of 16 lanes, then the rows' totals broadcast upwards
// to the last lane -- register traffic only, where a butterfly of shuffles goes through LDS six times.
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp_add(float v) {
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, ROWS, 0xF, false));
}
__device__ __forceinline__ float row16_sum(float v) {        // every lane: the sum of its row of 16
    v = dpp_add<0x128, 0xF>(v);                              // row_ror:8
    v = dpp_add<0x124, 0xF>(v);
    v = dpp_add<0x122, 0xF>(v);
    return dpp_add<0x121, 0xF>(v);
}
__device__ __forceinline__ float wave_sum(float v) {
    v = row16_sum(v);
    v = dpp_add<0x142, 0xA>(v);                              // row_bcast:15 into rows 1 and 3
    v = dpp_add<0x143, 0xC>(v);                              // row_bcast:31 into rows 2 and 3
    return __int_as_float(read_lane(__float_as_int(v), kWave - 1));
}

__device__ __forceinline__ float bf16_bits_to_f32(uint32_t b) { return __uint_as_float(b << 16); }

__device__ __forceinline__ uint32_t f32_to_bf16_bits(float f) {
    uint32_t u = __float_as_uint(f);
    if ((u & 0x7FFFFFFFu) > 0x7F800000u) return (u >> 16) | 0x0040u;        // quiet NaN
    return (u + 0x7FFFu + ((u >> 16) & 1u)) >> 16;                          // nearest even
}

// e4m3 "fn" (bias 7, no infinities) -> fp32, exact.
__device__ __forceinline__ float e4m3_to_f32(uint32_t c) {
    const uint32_t sign = (c & 0x80u) << 24;
    const uint32_t e = (c >> 3) & 0xFu, m = c & 0x7u;
    float mag = e ? __uint_as_float(((e + 120u) << 23) | (m << 20)) : (float)m * 0x1p-9f;
    if (e == 0xFu && m == 0x7u) mag = __uint_as_float(0x7FC00000u);
    return __uint_as_float(__float_as_uint(mag) | sign);
}

// N consecutive elements of a float row as fp32, and back with one rounding (to nearest even) each.  N = 8: `row` and
// `at` on 16-byte boundaries, moved as 16-byte vectors; N = 1: any alignment the element type has.
template <int DT, int N>
__device__ __forceinline__ void load_floats(const void *row, int64_t at, float *f) {
    static_assert(N == 1 || N == 8, "one element or one vector of eight");
    if constexpr (DT == TERRACE_F32) {
        if constexpr (N == 1) {
            f[0] = ((const float *)row)[at];
        } else {
            const u32x4 *p = (const u32x4 *)((const float *)row + at);
            const u32x4 a = ld_stream(p), b = ld_stream(p + 1);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                f[i] = __uint_as_float(a[i]);
                f[4 + i] = __uint_as_float(b[i]);
            }
        }
    } else {
        uint32_t bits[N == 1 ? 1 : 4];
        if constexpr (N == 1) {
            bits[0] = ((const uint16_t *)row)[at];
        } else {
            const u32x4 a = ld_stream((const u32x4 *)((const uint16_t *)row + at));
#pragma unroll
            for (int i = 0; i < 4; ++i) bits[i] = a[i];
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t b = i & 1 ? bits[i / 2] >> 16 : bits[i / 2] & 0xFFFFu;
            if constexpr (DT == TERRACE_BF16) f[i] = bf16_bits_to_f32(b);
            else f[i] = __half2float(__ushort_as_half((unsigned short)b));
        }
    }
}
// Two floats rounded (nearest even) to the halves of a register; bf16 pairs are one instruction on this part.
template <int DT>
__device__ __forceinline__ uint32_t to_bits16x2(float lo, float hi) {
    if constexpr (DT == TERRACE_BF16) {
        typedef float f32x2_t __attribute__((ext_vector_type(2)));
        typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t{lo, hi}), bf16x2_t));
    } else {
        return (uint32_t)__half_as_ushort(__float2half_rn(lo)) | ((uint32_t)__half_as_ushort(__float2half_rn(hi)) << 16);
    }
}
template <int DT>
__device__ __forceinline__ uint32_t to_bits16(float f) { return to_bits16x2<DT>(f, 0.0f) & 0xFFFFu; }
template <int DT, int N>
__device__ __forceinline__ void store_floats(void *row, int64_t at, const float *f) {
    static_assert(N == 1 || N == 8, "one element or one vector of eight");
    if constexpr (DT == TERRACE_F32) {
        if constexpr (N == 1) {
            ((float *)row)[at] = f[0];
        } else {
            u32x4 *p = (u32x4 *)((float *)row + at);
            u32x4 a, b;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                a[i] = __float_as_uint(f[i]);
                b[i] = __float_as_uint(f[4 + i]);
            }
            st_stream(p, a);
            st_stream(p + 1, b);
        }
    } else if constexpr (N == 1) {
        ((uint16_t *)row)[at] = (uint16_t)to_bits16<DT>(f[0]);
    } else {
        u32x4 a;
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = to_bits16x2<DT>(f[2 * i], f[2 * i + 1]);
        st_stream((u32x4 *)((uint16_t *)row + at), a);
    }
}

// A row-width argument of the C ABI may carry a pitch (TERRACE_ROW_PITCHED): `width` bytes of data every `pitch`
// bytes.  Packed rows have pitch == width.
struct RowGeom {
    int64_t width, pitch;
    bool pitched() const { return pitch != width; }
};
inline RowGeom row_geom(int64_t row_bytes) {
    RowGeom g{row_bytes & 0xFFFFFFFFll, row_bytes >> 32};
    if (g.pitch == 0) g.pitch = g.width;
    return g;
}
// Pitched rows move through the kilobyte-sliced kernels only: 16-byte-multiple widths on a whole number of
// kilobytes.  (The buffers must also be 16-byte aligned; the launchers check that.)
inline bool row_geom_ok(const RowGeom &g) {
    if (g.width < 0 || g.pitch < g.width) return false;
    return !g.pitched() || (g.width % 16 == 0 && g.pitch % 1024 == 0);
}

inline int check_launch() { return hipGetLastError() == hipSuccess ? TERRACE_OK : TERRACE_ELAUNCH; }

inline size_t align_up(size_t v, size_t a) { return (v + a - 1) / a * a; }

}  // namespace terrace

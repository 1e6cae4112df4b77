// nn_common.h -- element types, conversions, matrix instructions and guarded loads of the network-side operators (include/umr_nn.h).
#pragma once
#include "umr_common.h"
#include "../../include/umr_nn.h"

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// the bits of one as the other; by value (a bit cast straight from a vector's element is not one)
__device__ __forceinline__ float as_f32(unsigned u) { return __builtin_bit_cast(float, u); }
__device__ __forceinline__ unsigned as_u32(float f) { return __builtin_bit_cast(unsigned, f); }

struct bf16_t { unsigned short bits; };      // bfloat16 and half as their bits: arithmetic is done in fp32 or by the matrix unit
struct f16_t { unsigned short bits; };

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(bf16_t v) { return as_f32((unsigned)v.bits << 16); }
__device__ __forceinline__ float to_f32(f16_t v) { return (float)__builtin_bit_cast(_Float16, v.bits); }

// rounding to nearest even; the one rounding of a result that was held in fp32
template <class T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ f16_t from_f32<f16_t>(float v) { return f16_t{__builtin_bit_cast(unsigned short, (_Float16)v)}; }
template <> __device__ __forceinline__ bf16_t from_f32<bf16_t>(float v) {
#ifdef UMR_HOST_SHIM
    const unsigned u = __builtin_bit_cast(unsigned, v);
    if ((u & 0x7fffffffu) > 0x7f800000u) return bf16_t{(unsigned short)((u >> 16) | 64u)};
    return bf16_t{(unsigned short)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16)};
#else
    return bf16_t{__builtin_bit_cast(unsigned short, (__bf16)v)};      // v_cvt_pk_bf16_f32
#endif
}

// Matrix instructions.  Operand layout (lane l): the 32-row forms hold row l % 32, the 16-row forms row l % 16, of both operands
// and one 16-byte chunk of their contraction.  Which contraction index sits where does not matter as long as both operands agree:
// an fp32 chunk (4 values) is fed as 4 instructions of one value per lane, a 16-bit chunk (8 values) as one.
// Result (register r): column l % 32 of operand b, row 8 (r / 4) + 4 (l / 32) + r % 4 of operand a; the 16-row forms: column
// l % 16, row 4 (l / 16) + r.  With a = the operand whose rows run along memory in the result, a lane holds 4 neighbours.
#ifndef UMR_HOST_SHIM
__device__ __forceinline__ f32x16 mma32(float, u32x4 a, u32x4 b, f32x16 c) {
    const f32x4 af = __builtin_bit_cast(f32x4, a), bf = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_32x32x2f32(af[s], bf[s], c, 0, 0, 0);
    return c;
}
__device__ __forceinline__ f32x4 mma16(float, u32x4 a, u32x4 b, f32x4 c) {
    const f32x4 af = __builtin_bit_cast(f32x4, a), bf = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_16x16x4f32(af[s], bf[s], c, 0, 0, 0);
    return c;
}
typedef __bf16 bf16x8_v __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_v __attribute__((ext_vector_type(8)));
__device__ __forceinline__ f32x16 mma32(bf16_t, u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_v, a), __builtin_bit_cast(bf16x8_v, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma32(f16_t, u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_v, a), __builtin_bit_cast(f16x8_v, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma16(bf16_t, u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_v, a), __builtin_bit_cast(bf16x8_v, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma16(f16_t, u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_v, a), __builtin_bit_cast(f16x8_v, b), c, 0, 0, 0);
}
#else       // defined by the tests' emulation build (tests/host_kernel/nn_tu.cpp)
template <class T> f32x16 mma32(T, u32x4 a, u32x4 b, f32x16 c);
template <class T> f32x4 mma16(T, u32x4 a, u32x4 b, f32x4 c);
#endif

// Steps of a butterfly over the 2, 4 .. 64 lanes of a row: the partner's value, where a step may take any lane of the partner's group
// because the groups of O lanes already agree (O = 4, 8: the mirrored lane).  Up to 16 lanes these are DPP moves, without LDS.
template <int O> __device__ __forceinline__ float across(float v) {
#ifndef UMR_HOST_SHIM
    constexpr int ctrl = O == 1 ? 0xB1 /* quad_perm 1,0,3,2 */ : O == 2 ? 0x4E /* 2,3,0,1 */ : O == 4 ? 0x141 /* half mirror */ : 0x140 /* mirror */;
    if constexpr (O <= 8) return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), ctrl, 0xf, 0xf, true));
#endif
    return __shfl_xor(v, O, UMR_WAVE);
}
template <int N> __device__ __forceinline__ float group_sum(float v) {          // over groups of N lanes; every lane gets it
    if constexpr (N >= 2) v += across<1>(v);
    if constexpr (N >= 4) v += across<2>(v);
    if constexpr (N >= 8) v += across<4>(v);
    if constexpr (N >= 16) v += across<8>(v);
    if constexpr (N >= 32) v += across<16>(v);
    if constexpr (N >= 64) v += across<32>(v);
    return v;
}
template <int N> __device__ __forceinline__ float group_max(float v) {          // NaN is left out
    if constexpr (N >= 2) v = fmaxf(v, across<1>(v));
    if constexpr (N >= 4) v = fmaxf(v, across<2>(v));
    if constexpr (N >= 8) v = fmaxf(v, across<4>(v));
    if constexpr (N >= 16) v = fmaxf(v, across<8>(v));
    if constexpr (N >= 32) v = fmaxf(v, across<16>(v));
    if constexpr (N >= 64) v = fmaxf(v, across<32>(v));
    return v;
}
__device__ __forceinline__ float exp2_of(float x) {      // one v_exp_f32: results below 2^-126 are 0
#ifndef UMR_HOST_SHIM
    return __builtin_amdgcn_exp2f(x);
#else
    return exp2f(x);
#endif
}

// Nothing is scheduled across: loads that were written ahead of the matrix instructions stay ahead of them.
#ifndef UMR_HOST_SHIM
#define UMR_SCHED_FENCE() __builtin_amdgcn_sched_barrier(0)
#else
#define UMR_SCHED_FENCE() ((void)0)
#endif

// Loads at the element's own alignment: this target's global loads take any, so rows of odd length need no other kernel.
typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef u32x2 u32x2_any __attribute__((aligned(2)));
typedef unsigned u32_any __attribute__((aligned(2)));
template <class T> __device__ __forceinline__ u32x4 load16B(const T *p) { return *(const u32x4_any *)p; }
// the first n of 16 / sizeof(T) elements at p, zeros behind them; nothing is read for n <= 0
template <class T> __device__ __forceinline__ u32x4 load16B_n(const T *p, long n) {
    constexpr int V = 16 / (int)sizeof(T);
    if (n >= V) return load16B(p);
    u32x4 r = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (i < n) {
            if constexpr (sizeof(T) == 4) r[i] = as_u32(p[i]);
            else r[i / 2] |= (unsigned)p[i].bits << (16 * (i & 1));
        }
    return r;
}
template <class T> __device__ __forceinline__ float elem_of(u32x4 v, int i) {     // element i of a loaded chunk, as fp32
    if constexpr (sizeof(T) == 4) return as_f32(v[i]);
    else return to_f32(T{(unsigned short)(v[i / 2] >> (16 * (i & 1)))});
}

// 4 neighbouring elements (fewer at an edge): loads to fp32 and stores from it
template <class T> __device__ __forceinline__ void load4(const T *p, long n, float (&v)[4]) {
    if (n >= 4) {
        if constexpr (sizeof(T) == 4) {
            const u32x4 r = *(const u32x4_any *)p;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = as_f32(r[i]);
        } else {
            const u32x2 r = *(const u32x2_any *)p;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = to_f32(T{(unsigned short)(r[i / 2] >> (16 * (i & 1)))});
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = i < n ? to_f32(p[i]) : 0.f;
    }
}
template <class T> __device__ __forceinline__ void store4(T *p, long n, const float (&v)[4]) {
    if (n >= 4) {
        if constexpr (sizeof(T) == 4) {
            u32x4 r;
#pragma unroll
            for (int i = 0; i < 4; ++i) r[i] = as_u32(v[i]);
            *(u32x4_any *)p = r;
        } else {
            u32x2 r;
#pragma unroll
            for (int i = 0; i < 2; ++i) r[i] = (unsigned)from_f32<T>(v[2 * i]).bits | ((unsigned)from_f32<T>(v[2 * i + 1]).bits << 16);
            *(u32x2_any *)p = r;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < n) p[i] = from_f32<T>(v[i]);
    }
}

// 4 bytes of a result; STREAM: past the caches
template <bool STREAM, class T> __device__ __forceinline__ void store_word(T *p, unsigned v) {
#ifndef UMR_HOST_SHIM
    if constexpr (STREAM) { __builtin_nontemporal_store(v, (u32_any *)p); return; }
#endif
    *(u32_any *)p = v;
}

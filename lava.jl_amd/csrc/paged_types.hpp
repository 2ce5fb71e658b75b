// paged_types.hpp -- the two operand types of the paged attention kernels, and small device helpers (internal).
#pragma once
#include <hip/hip_runtime.h>

#include "lava_coopmat.hpp"

namespace lava {

template <int N>
struct pg_int {
    static constexpr int value = N;
};
template <bool B>
struct pg_tag {
    static constexpr bool value = B;
};

typedef short pg_s16x4 __attribute__((ext_vector_type(4)));

template <typename T>
struct PgType;
template <>
struct PgType<f16> {
    typedef f16x8 v8;
    typedef f16x4 v4;
    typedef f16 v2 __attribute__((ext_vector_type(2)));
    __device__ static f32x4 mma16(v8 a, v8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
    __device__ static f32x16 mma32(v8 a, v8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
    // x + the two values
    __device__ static float dot2(v2 a, float x) {
        const v2 ones = {(f16)1.f, (f16)1.f};
        return __builtin_amdgcn_fdot2(a, ones, x, false);
    }
};
template <>
struct PgType<bf16> {
    typedef bf16x8 v8;
    typedef bf16x4 v4;
    typedef bf16 v2 __attribute__((ext_vector_type(2)));
    __device__ static f32x4 mma16(v8 a, v8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
    __device__ static f32x16 mma32(v8 a, v8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
    __device__ static float dot2(v2 a, float x) {
        const v2 ones = {(bf16)1.f, (bf16)1.f};
        return __builtin_amdgcn_fdot2_f32_bf16(a, ones, x, false);
    }
};

// Values that are not finite, at keys that only some rows of a tile see: P V is a matrix product and 0 times infinity is
// NaN, in rows that do not see the key.  Where a tile of values has any, they enter as zeros, and what they are worth to
// each row comes from products of where they are with which keys the row sees -- not with P, whose weight for a key may be below all
// numbers of the type (f16: a score 17 below the row's largest), where a value that the row sees would vanish.

typedef uint16_t pg_u16x2 __attribute__((ext_vector_type(2)));
typedef uint16_t pg_u16x8 __attribute__((ext_vector_type(8)));
template <typename T>
constexpr uint16_t PG_EXPONENT = sizeof(T) == 2 && __is_same(T, bf16) ? 0x7f80 : 0x7c00;

// Whether one of `bytes` bytes of LDS from `at` on is of a value that is not finite (by a wavefront together, 1024 at a time).
template <typename T, int BYTES>
__device__ __forceinline__ bool pg_not_finite(uint32_t at, int lane) {
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) const u4 lds_u4;
    pg_u16x2 top = {0, 0};
#pragma unroll 8
    for (int i = 0; i < BYTES / 1024; ++i) {
        const u4 u = *(lds_u4*)(uintptr_t)(at + 16u * (uint32_t)lane + 1024u * (uint32_t)i);
#pragma unroll
        for (int k = 0; k < 4; ++k) top = __builtin_elementwise_max(top, __builtin_bit_cast(pg_u16x2, u[k] & 0x7fff7fffu));
    }
    return __builtin_amdgcn_ballot_w64(max(top[0], top[1]) >= PG_EXPONENT<T>) != 0;
}

// 0 in place of such values there.
template <typename T, int BYTES>
__device__ __forceinline__ void pg_drop_not_finite(uint32_t at, int lane) {
    typedef __attribute__((address_space(3))) pg_u16x8 lds_u16x8;
#pragma unroll 1
    for (int i = 0; i < BYTES / 1024; ++i) {
        lds_u16x8* const x = (lds_u16x8*)(uintptr_t)(at + 16u * (uint32_t)lane + 1024u * (uint32_t)i);
        pg_u16x8 v = *x;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (v[e] & 0x7fff) >= PG_EXPONENT<T> ? (uint16_t)0 : v[e];
        *x = v;
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
}

// 1 where a is +infinity or NaN (up), where it is -infinity or NaN (down).  Returns a with 0 in their place.
template <typename T, typename V>
__device__ __forceinline__ V pg_split(V a, V& up, V& down) {
    pg_u16x8 x = __builtin_bit_cast(pg_u16x8, a);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const uint16_t b = x[e] & 0x7fff;
        const bool off = b >= PG_EXPONENT<T>, nan = b > PG_EXPONENT<T>, minus = (x[e] >> 15) != 0;
        up[e] = off && (nan || !minus) ? (T)1.f : (T)0.f;
        down[e] = off && (nan || minus) ? (T)1.f : (T)0.f;
        x[e] = off ? (uint16_t)0 : x[e];
    }
    return __builtin_bit_cast(V, x);
}

// 1 for the keys that a row sees, from P with -0 for masked ones.
template <typename T, typename V>
__device__ __forceinline__ V pg_seen(V p) {
    constexpr uint16_t one = __is_same(T, bf16) ? 0x3f80 : 0x3c00;
    pg_u16x8 x = __builtin_bit_cast(pg_u16x8, p);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = x[e] == 0x8000 ? (uint16_t)0 : one;
    return __builtin_bit_cast(V, x);
}

// What infinities of the sign add to the sums o where `count` of them lie at keys that the row sees: infinite for every count but 0.
template <typename F>
__device__ __forceinline__ void pg_add_not_finite(F& o, const F& count, float sign) {
#pragma unroll
    for (int r = 0; r < (int)(sizeof(F) / 4); ++r) {
#pragma clang fp contract(off)   // a fused product would stay finite, and infinity minus it infinite
        const float x = count[r] * 0x1p127f * (sign * 0x1p127f);
        o[r] = o[r] + x;
    }
}

// x of lanes 0-31 and of lanes 32-63, to all (two copies of x: one register swapped with itself gives no halves)
__device__ __forceinline__ void pg_xor32_pair(float x, float& a, float& b) {
    a = x;
    b = x;
    asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b));
}

}  // namespace lava

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

// q = f16(q c) in place, rounded once: the mixed-precision FMA on either half of a register.  The s_nop is for
// an MFMA that reads q next.  (bf16 has no such instruction, and no use for it: one rounding of q c would cost 2^-8.)
__device__ __forceinline__ void pg_scale_f16(f16x8& q, float c) {
    uint4 u = __builtin_bit_cast(uint4, q);
    asm("v_fma_mixlo_f16 %0, %0, %4, 0 op_sel_hi:[1,0,0]\n\t"
        "v_fma_mixhi_f16 %0, %0, %4, 0 op_sel:[1,0,0] op_sel_hi:[1,0,0]\n\t"
        "v_fma_mixlo_f16 %1, %1, %4, 0 op_sel_hi:[1,0,0]\n\t"
        "v_fma_mixhi_f16 %1, %1, %4, 0 op_sel:[1,0,0] op_sel_hi:[1,0,0]\n\t"
        "v_fma_mixlo_f16 %2, %2, %4, 0 op_sel_hi:[1,0,0]\n\t"
        "v_fma_mixhi_f16 %2, %2, %4, 0 op_sel:[1,0,0] op_sel_hi:[1,0,0]\n\t"
        "v_fma_mixlo_f16 %3, %3, %4, 0 op_sel_hi:[1,0,0]\n\t"
        "v_fma_mixhi_f16 %3, %3, %4, 0 op_sel:[1,0,0] op_sel_hi:[1,0,0]\n\t"
        "s_nop 1"
        : "+v"(u.x), "+v"(u.y), "+v"(u.z), "+v"(u.w)
        : "v"(c));
    q = __builtin_bit_cast(f16x8, u);
}

// x of lanes 0-31 and of lanes 32-63, to all (two copies of x: one register swapped with itself gives no halves)
__device__ __forceinline__ void pg_xor32_pair(float x, float& a, float& b) {
    a = x;
    b = x;
    asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b));
}

}  // namespace lava

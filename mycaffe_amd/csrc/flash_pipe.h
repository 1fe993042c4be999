// What the kernels with a software pipeline inside the wavefront share (attn_flash2.hip, attn_paged_pipe.hip): exchanges between the two halves
// of a row, pairs of weights, and the pinned matrix instructions.
#pragma once
#include "flash_traits.h"

namespace mch {

__device__ __forceinline__ float f2_pair_sum(float v)   // v + the value of the lane 32 away; both lanes get the same bits
{
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float f2_pair_max(float v)
{
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float f2_dot2_ones(uint32_t pair, float acc)   // acc + lo(pair) + hi(pair), bf16 pair
{
    const bf16x2 ones = {(__bf16)1.0f, (__bf16)1.0f};
    return __builtin_amdgcn_fdot2_f32_bf16(*reinterpret_cast<bf16x2*>(&pair), ones, acc, false);
}
__device__ __forceinline__ uint32_t f2_pack_trunc(float lo, float hi)   // the upper halves of two floats: a bf16 pair
{
    // Rounding towards zero: the row sums are formed from these same pairs, so the one-sided error cancels between the
    // weights and their sum, and v_perm_b32 runs at the full rate where the rounding conversion runs at half of it.
    return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
}
// MFMAs of the pinned phases.  "v": vector register, "a": accumulation register.  The compiler cannot see into the
// assembly, so the distances the hardware wants around an MFMA are kept by the order the phases are written in: two
// MFMAs that accumulate onto the same tile are at least one other MFMA apart, and a tile's first other reader is at
// least four MFMAs after its last writer.
__device__ __forceinline__ void f2_mma_s_first(floatx16& d, const u32x4& k, const u32x4& q)   // d (v) = K (v) Q^T (a)
{
    asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, 0" : "=&v"(d) : "v"(k), "a"(q));
}
__device__ __forceinline__ void f2_mma_s_acc(floatx16& d, const u32x4& k, const u32x4& q)
{
    asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(d) : "v"(k), "a"(q));
}
__device__ __forceinline__ void f2_mma_o_acc(floatx16& o, const u32x4& vt, const u32x4& p)    // o (a) += V^T (v) P^T (v)
{
    asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+a"(o) : "v"(vt), "v"(p));
}

}  // namespace mch

// Operands of the attention kernels' 16 x 16 tiles: the matrix instruction, probabilities rounded to the query's type, e4m3 codes widened to it.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace pto_hip {
namespace attn {

typedef __attribute__((__vector_size__(4 * sizeof(float)))) float f32x4;
typedef __attribute__((__vector_size__(4 * sizeof(uint32_t)))) uint32_t u32x4;
typedef __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16 bf16x8;
typedef __attribute__((__vector_size__(8 * sizeof(_Float16)))) _Float16 f16x8;

template <bool BF16>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (BF16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
}

// Round two fp32 to the 16-bit activation type (nearest even) and pack; also returns the
// rounded values so the row sum is taken over exactly what the PV product sees
// (04_paged_attention.py:98-100).
template <bool BF16>
__device__ __forceinline__ uint32_t round_pack(float a, float b, float& ra, float& rb) {
  if constexpr (BF16) {
    __bf16 x = (__bf16)a, y = (__bf16)b;
    ra = (float)x;
    rb = (float)y;
    return (uint32_t)__builtin_bit_cast(uint16_t, x) |
           ((uint32_t)__builtin_bit_cast(uint16_t, y) << 16);
  } else {
    _Float16 x = (_Float16)a, y = (_Float16)b;
    ra = (float)x;
    rb = (float)y;
    return (uint32_t)__builtin_bit_cast(uint16_t, x) |
           ((uint32_t)__builtin_bit_cast(uint16_t, y) << 16);
  }
}

// Two e4m3 codes (low or high half of a dword) -> two packed bf16 or fp16 values; both types
// hold every e4m3 value exactly.
template <bool BF16>
__device__ __forceinline__ uint32_t fp8x2_widen(uint32_t w, bool hi) {
  if constexpr (BF16) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const bf16x2 r = hi ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true)
                        : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false);
    return __builtin_bit_cast(uint32_t, r);
  } else {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    const f16x2 r = hi ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true)
                       : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false);
    return __builtin_bit_cast(uint32_t, r);
  }
}
template <bool BF16>
__device__ __forceinline__ u32x4 fp8x8_widen(uint32_t w0, uint32_t w1) {
  return u32x4{fp8x2_widen<BF16>(w0, false), fp8x2_widen<BF16>(w0, true), fp8x2_widen<BF16>(w1, false),
               fp8x2_widen<BF16>(w1, true)};
}

}  // namespace attn
}  // namespace pto_hip

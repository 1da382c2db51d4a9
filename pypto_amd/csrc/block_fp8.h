// e4m3 codes with a scale for each block of 128: what the kernels on such operands share.
//
// An activation row carries one fp32 scale per 128 columns ([rows, ceil(cols / 128)], row-major), a weight matrix, stored
// one row per OUTPUT channel with k contiguous ([n, k]), one per block of 128 x 128 ([ceil(n / 128), ceil(k / 128)]); a value is its code
// times its scale.  The scale of a group is amax / 448, so that its largest element meets the format's largest value.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace pto_hip {
namespace block8 {

constexpr int kBlock = 128;  // elements that share a scale
constexpr int kMaxK = 65536;  // longest rows of the products: byte offsets inside a tile stay far below 2^31

// Whether two ranges of bytes have any in common (null: none).
inline bool overlap(const void* a, int64_t a_bytes, const void* b, int64_t b_bytes) {
  const uintptr_t pa = (uintptr_t)a, pb = (uintptr_t)b;
  return a && b && pa < pb + (uintptr_t)b_bytes && pb < pa + (uintptr_t)a_bytes;
}

typedef __attribute__((__vector_size__(4 * sizeof(float)))) float f32x4;
typedef __attribute__((__vector_size__(4 * sizeof(int)))) int i32x4;

template <int N>
struct IntConst {
  static constexpr int value = N;
};

// Scale of a group whose largest magnitude is amax: 1 for a group of zeros, and never below the smallest normal number (whose
// reciprocal is one too).
__device__ __forceinline__ float group_scale(float amax) { return amax > 0.f ? fmaxf(amax / 448.f, 0x1p-126f) : 1.f; }

// The size of a finite value, 0 of others.
__device__ __forceinline__ float finite_size(float v) { return fabsf(v) <= 3.4028234664e38f ? fabsf(v) : 0.f; }
// The power of two that, divided out, puts a largest size of amax into [2^14, 2^15); 0 for none, and within what fp32 holds.
__device__ __forceinline__ int half_exponent(float amax) { return amax > 0.f ? max(ilogbf(amax) - 14, -126) : 0; }

// v / scale as often as a group has elements.
struct GroupQuotient {
  float s, r;
  __device__ __forceinline__ explicit GroupQuotient(float scale) : s(scale) {
    r = __builtin_amdgcn_rcpf(s);
    r = fmaf(fmaf(-s, r, 1.f), r, r);
  }
  // Correctly rounded: the reciprocal is refined once to half an ulp, the quotient twice by its exact remainder (as in ffn_fp8.hip's row
  // quantiser).  No quotient of a finite group leaves +-448 (1 + 2^-23), which rounds to a code without a clamp; an infinite scale (an infinite
  // element) takes the division itself.
  __device__ __forceinline__ float operator()(float v) const {
    if (__builtin_expect(!(s <= 3.4028234664e38f), 0)) return v / s;
    const float q0 = v * r;
    const float q1 = fmaf(fmaf(-q0, s, v), r, q0);
    const float q2 = fmaf(fmaf(-q1, s, v), r, q1);
    return v == 0.f ? v : q2;  // a zero keeps its sign
  }
  // Within an ulp and a half, for values that are further off themselves (h, whose exponential and reciprocal are off by 2^-17); of an
  // infinite scale the same as the division, zeros and NaN.
  __device__ __forceinline__ float near(float v) const { return v * (s <= 3.4028234664e38f ? r : 0.f); }
};

// Four quotients as codes, the first in the lowest byte (round to nearest even; NaN stays NaN).
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
  return (uint32_t)w;
}

}  // namespace block8
}  // namespace pto_hip

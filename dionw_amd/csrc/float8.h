// Shared by the 8-bit matrices' kernels: the format, and how much of it a product needs.
#pragma once

#include "common.h"

namespace dionw {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

constexpr int kTile = 128;  // columns (and rows) that share a scale

// The scale's exponent byte of a block whose largest finite magnitude has the bits `largest`
// (at least 1: the scale and its reciprocal are normal).
__device__ __forceinline__ uint32_t scale_byte(uint32_t largest) {
  const uint32_t field = (largest + 0x1FFFFFu) >> 23;  // fractions above 1.75 carry
  return field > 8u ? field - 8u : 1u;
}
__device__ __forceinline__ float power(uint32_t byte) { return __uint_as_float(byte << 23); }

// The bits of |v|, 0 where it is not finite (such values become NaN codes and leave the
// block's scale alone).
__device__ __forceinline__ uint32_t magnitude(float v) {
  const uint32_t b = __float_as_uint(v) & 0x7FFFFFFFu;
  return b < 0x7F800000u ? b : 0u;
}

// Four codes of four values, rounded to nearest even; infinities become NaN.
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d, float inv) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a * inv, b * inv, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c * inv, d * inv, w, true);
}

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(_Float16 v) { return (float)v; }
__device__ __forceinline__ float to_float(__bf16 v) { return (float)v; }

// Codes are expanded to bfloat16 with half their scale, as 448 x 2^120 (what a block of
// magnitudes up to the largest float32 may round to) is past bfloat16. Sums of products of
// two expanded operands take kExpanded back.
__device__ __forceinline__ float half_power(uint32_t byte) { return __uint_as_float((byte - 1) << 23); }
constexpr float kExpanded = 4.f;

// Eight codes and their scale as bfloat16, exactly (a code has 4 significant bits).
__device__ __forceinline__ bf16x8 expand(uint32_t lo, uint32_t hi, float scale) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
  return __builtin_shufflevector(__builtin_shufflevector(a, b, 0, 1, 2, 3),
                                 __builtin_shufflevector(c, d, 0, 1, 2, 3), 0, 1, 2, 3, 4, 5, 6, 7);
}

}  // namespace dionw

// Shared by the 4-bit matrices' kernels: the format, and how values are rounded to it.
#pragma once

#include "float8.h"

namespace dionw {

typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr int kBlock4 = 32;    // columns (and rows) that share a scale
constexpr int kDepth4 = 256;   // a matrix's rows run to a multiple: 128 bytes, one stage of a product

// A 4-bit matrix: rows of depth / 2 bytes, one behind the other; data null: nothing.
using Matrix4 = Matrix;

// The random bits of a stochastic rounding: a seed, or where it lies in device memory.
struct Noise {
  int64_t seed;
  const int64_t* at;
};

// What dionw_float4_quantize does to one matrix.
struct Quantization4 {
  int32_t elem;
  const void* x;
  int64_t rows, cols, ld;
  Matrix4 by_row, by_col;
  float* sums;
};
int quantize4(const Quantization4& x, bool tiles, const Noise* noise, hipStream_t stream);
// x by rows and columns and w by tiles, in one launch.
int quantize4_pair(const Quantization4& x, const Quantization4& w, hipStream_t stream);

// The exponent byte of the scale of a block whose largest magnitude has the bits `largest`: the
// smallest power of two that brings it to 7 at most (what is above 6 then rounds to 6, half a step
// off at worst: on normal values this loses 3% less than scaling to 6), or, rounded stochastically,
// to 6 (above it every value would be rounded down). At least 1: the scale and its reciprocal are
// normal. A block that holds an infinity or NaN gets 255, which makes all of it NaN: codes cannot.
template <bool STOCHASTIC>
__device__ __forceinline__ uint32_t scale_byte4(uint32_t largest) {
  const uint32_t field = (largest + (STOCHASTIC ? 0x3FFFFFu : 0x1FFFFFu)) >> 23;
  return largest >= 0x7F800000u ? 255u : field > 2u ? field - 2u : 1u;
}
// 1 / scale (of a scale of 255: of anything finite).
__device__ __forceinline__ float inverse4(uint32_t byte) { return power(byte < 254u ? 254u - byte : 1u); }

// Two rounds of multiply and xor-shift.
__device__ __forceinline__ uint32_t mix32(uint32_t x) {
  x ^= x >> 16;
  x *= 0x9E3779B1u;
  x ^= x >> 15;
  x *= 0x85EBCA77u;
  return x ^ (x >> 16);
}
__device__ __forceinline__ uint32_t noise_key(const Noise& n) {
  const uint64_t seed = n.at ? (uint64_t)*n.at : (uint64_t)n.seed;
  return mix32((uint32_t)seed + 0x9E3779B1u * ((uint32_t)(seed >> 32) + 1u));
}
// 22 bits each for an even column's value and the next one's, from a pair's 32.
__device__ __forceinline__ uint32_t even_noise(uint32_t h) { return h >> 10; }
__device__ __forceinline__ uint32_t odd_noise(uint32_t h) { return (h & 0xFFFFu) << 6; }

// x / scale rounded up by `noise` of 2^22, down otherwise, as a value of the format. From 1 on the
// format keeps one fraction bit of a value, so the noise is added below it and what is below it
// dropped; 1 is added to smaller values first, whose steps are those of the next binade
// (which rounds them to a multiple of 2^-23).
__device__ __forceinline__ float stochastic4(float x, float scale, float inverse, uint32_t noise) {
  const float one = __builtin_copysignf(fabsf(x) < scale ? 1.f : 0.f, x);
  const uint32_t w = __float_as_uint(__builtin_fmaf(x, inverse, one)) + noise;
  return __uint_as_float(w & 0xFFC00000u) - one;
}

// Codes of two values times 1 / scale, rounded to nearest (ties to the even code) and cut at 6, in
// byte B of `old`; the first value's in its low half.
template <int B>
__device__ __forceinline__ uint32_t codes2(uint32_t old, uint32_t pair, float scale, __bf16) {
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(old, __builtin_bit_cast(bf16x2, pair), scale, B);
}
template <int B>
__device__ __forceinline__ uint32_t codes2(uint32_t old, uint32_t pair, float scale, _Float16) {
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(old, __builtin_bit_cast(f16x2, pair), scale, B);
}
template <int B>
__device__ __forceinline__ uint32_t codes2(uint32_t old, float a, float b, float scale) {
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(old, a, b, scale, B);
}

// The largest over 4 adjacent lanes.
__device__ __forceinline__ uint32_t largest_of_four(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, false));
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, false));
}

}  // namespace dionw

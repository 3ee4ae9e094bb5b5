// Shared by the 4-bit matrices' kernels: the format, and how values are rounded to it.
#pragma once

#include "float8.h"

namespace dionw {

typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr int kBlock4 = 32;   // columns (and rows) that share a scale
constexpr int kDepth4 = 256;  // a matrix's rows run to a multiple: 128 bytes, one stage of a product

constexpr int kTile4 = 128;   // side of a quantization's tiles; rows that share partial column sums

// A 4-bit matrix: rows of depth / 2 bytes, one behind the other; data null: nothing.
using Matrix4 = Matrix;

// The random bits of a stochastic rounding: a seed, or where it lies in device memory. Of a pair of
// columns' 32 bits the even one's value takes the top 22, the odd one's the low 16.
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
// x / scale (6 at most), below 1 rounded to a multiple of 2^-23: what lies below the last place kept is
// then a multiple of 2^-22 of it, like the noise. float32: 1 is added and taken off. 16 bits: 1.5, whatever
// the sign and size, which takes an instruction less: a magnitude below 0.5 gives a sum from 1 to 2, whose last
// place is 2^-23 (1.5 is an even multiple of it, so that ties go where they belong); a larger one is a
// multiple of 2^-11 and stays exact in a sum below 8.
template <typename T>
__device__ __forceinline__ float scaled4(float x, float scale, float inverse) {
  const float one = sizeof(T) < 4 ? 1.5f : __builtin_copysignf(fabsf(x) < scale ? 1.f : 0.f, x);
  return __builtin_fmaf(x, inverse, one) - one;
}

// Codes of eight scaled values, rounded up by chance: `noise` holds each value's bits at the
// top of a word. The instruction takes two values and adds to the first one's part below the last
// place kept its third operand / 2^32 of that place, to the second's the same word turned left by
// one bit, and drops what is left of both; values below 1 lose what is below 2^-23 first (measured
// bit by bit; its 16-bit forms lose what is below 2^-7 and 2^-10, so float32 serves every type). A pair's
// bits are 22 and 16 of one word in places of their own, so that each of a pair's codes comes
// from an instruction of its own: the words' low halves (bits 0..3 of each byte) from `even`, the others from
// `odd`. In assembly, as the builtin leaves out that the destination's other bytes are kept; a
// byte's write needs one more instruction before the next one that keeps it, which the two words'
// turns are.
__device__ __forceinline__ uint32_t noisy8(const f32x2 (&p)[4], const uint32_t (&noise)[8]) {
  uint32_t even = 0, odd = 0;
#ifdef __HIP_DEVICE_COMPILE__
  asm("v_cvt_scalef32_sr_pk_fp4_f32 %0, %2, %6, %14\n\t"
      "v_cvt_scalef32_sr_pk_fp4_f32 %1, %2, %7, %14\n\t"
      "v_cvt_scalef32_sr_pk_fp4_f32 %0, %3, %8, %14 op_sel:[0,0,1,0]\n\t"
      "v_cvt_scalef32_sr_pk_fp4_f32 %1, %3, %9, %14 op_sel:[0,0,1,0]\n\t"
      "v_cvt_scalef32_sr_pk_fp4_f32 %0, %4, %10, %14 op_sel:[0,0,0,1]\n\t"
      "v_cvt_scalef32_sr_pk_fp4_f32 %1, %4, %11, %14 op_sel:[0,0,0,1]\n\t"
      "v_cvt_scalef32_sr_pk_fp4_f32 %0, %5, %12, %14 op_sel:[0,0,1,1]\n\t"
      "v_cvt_scalef32_sr_pk_fp4_f32 %1, %5, %13, %14 op_sel:[0,0,1,1]\n\t"
      "s_nop 0"
      : "=&v"(even), "=&v"(odd)
      : "v"(p[0]), "v"(p[1]), "v"(p[2]), "v"(p[3]), "v"(noise[0]), "v"(noise[1] >> 1), "v"(noise[2]),
        "v"(noise[3] >> 1), "v"(noise[4]), "v"(noise[5] >> 1), "v"(noise[6]), "v"(noise[7] >> 1), "v"(1.f));
#endif
  return (even & 0x0F0F0F0Fu) | (odd & 0xF0F0F0F0u);
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

// Codes of a row or a column of a Square times 1 / scale, to nearest.
template <typename T>
struct Codes {
  using S = Square<T>;
  template <int B>
  __device__ __forceinline__ static uint32_t row_pair(uint32_t old, const S& v, int i, float scale) {
    if constexpr (sizeof(T) == 4) return codes2<B>(old, v.value(i, 2 * B), v.value(i, 2 * B + 1), scale);
    else return codes2<B>(old, v.w[i][B], scale, T{});
  }
  template <int B>
  __device__ __forceinline__ static uint32_t col_pair(uint32_t old, const S& v, int k, float scale) {
    if constexpr (sizeof(T) == 4)
      return codes2<B>(old, v.value(2 * B, k), v.value(2 * B + 1, k), scale);
    else
      return codes2<B>(old, __builtin_amdgcn_perm(v.w[2 * B + 1][k >> 1], v.w[2 * B][k >> 1],
                                                  k & 1 ? 0x07060302u : 0x05040100u), scale, T{});
  }
  __device__ __forceinline__ static uint32_t row(const S& v, int i, float scale) {
    return row_pair<3>(row_pair<2>(row_pair<1>(row_pair<0>(0, v, i, scale), v, i, scale), v, i, scale), v, i, scale);
  }
  __device__ __forceinline__ static uint32_t col(const S& v, int k, float scale) {
    return col_pair<3>(col_pair<2>(col_pair<1>(col_pair<0>(0, v, k, scale), v, k, scale), v, k, scale), v, k, scale);
  }
};

// The largest over 4 adjacent lanes.
__device__ __forceinline__ uint32_t largest_of_four(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, false));
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, false));
}

}  // namespace dionw

// Shared by the 8-bit matrices' kernels: the format, and how much of it a product needs.
#pragma once

#include "common.h"

namespace dionw {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
// 16 bytes of a row that may start at any element: the hardware takes such loads whole.
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

constexpr int kTile = 128;  // columns (and rows) that share a scale
// A product's operand has rows of fewer bytes: a tile's rows are addressed with 32-bit offsets.
constexpr int64_t kRowBytes = 1 << 23;

// Codes with their scales, or (scale null) expanded codes; data null: nothing.
struct Matrix {
  void* data;
  void* scale;
  int64_t rows, depth, scale_ld;
};

// What dionw_float8_quantize does to one matrix.
struct Quantization {
  int32_t elem;
  const void* x;
  int64_t rows, cols, ld;
  Matrix by_row, by_col;
  float* sums;
};
// x by rows and columns and w by tiles, in one launch.
int quantize_pair(const Quantization& x, const Quantization& w, hipStream_t stream);
// x by rows and columns, and beside it, in the same launch, the codes of `from` expanded into `to`
// where it has room.
int quantize_and_expand(const Quantization& x, const Matrix (&from)[2], const Matrix (&to)[2],
                        hipStream_t stream);

// The scale's exponent byte of a block whose largest finite magnitude has the bits `largest`
// (at least 1: the scale and its reciprocal are normal).
__device__ __forceinline__ uint32_t scale_byte(uint32_t largest) {
  const uint32_t field = (largest + 0x1FFFFFu) >> 23;  // fractions above 1.75 carry
  return field > 8u ? field - 8u : 1u;
}
__device__ __forceinline__ float power(uint32_t byte) { return __uint_as_float(byte << 23); }

// Codes are expanded to bfloat16 with half their scale, as 448 x 2^120 (what a block of
// magnitudes up to the largest float32 may round to) is past bfloat16. Sums of products of
// two expanded operands take kExpanded back.
__device__ __forceinline__ float half_power(uint32_t byte) {
  return __uint_as_float((max(byte, 1u) - 1) << 23);  // exponent 0 scales by 2^-127
}
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

// Two values of a thread as they lie in memory: one word of 16-bit ones, two of float32.
template <typename T>
struct Pair;
template <typename T>
struct Pair16 {
  uint32_t w;
  // magnitudes, two 16-bit integers
  __device__ __forceinline__ uint32_t most() const { return w & 0x7FFF7FFFu; }
  __device__ __forceinline__ static uint32_t larger(uint32_t a, uint32_t b) {
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a),
                                                                  __builtin_bit_cast(u16x2, b)));
  }
};
template <>
struct Pair<__bf16> : Pair16<__bf16> {
  static constexpr uint32_t inf = 0x7F80u;
  __device__ __forceinline__ static uint32_t bits(uint32_t m) { return m << 16; }
  __device__ __forceinline__ float value(int k) const {
    return __uint_as_float(k ? w & 0xFFFF0000u : w << 16);
  }
};
template <>
struct Pair<_Float16> : Pair16<_Float16> {
  static constexpr uint32_t inf = 0x7C00u;
  __device__ __forceinline__ static uint32_t bits(uint32_t m) {
    return __float_as_uint((float)__builtin_bit_cast(_Float16, (uint16_t)m));
  }
  __device__ __forceinline__ float value(int k) const {
    return (float)__builtin_bit_cast(_Float16, (uint16_t)(k ? w >> 16 : w));
  }
};

typedef short i16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// Codes of four values times 1 / scale, rounded to nearest even; infinities become NaN.
__device__ __forceinline__ uint32_t codes4(uint32_t lo, uint32_t hi, float scale, __bf16) {
  i16x2 o = {0, 0};
  o = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(o, __builtin_bit_cast(bf16x2, lo), scale, false);
  o = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(o, __builtin_bit_cast(bf16x2, hi), scale, true);
  return __builtin_bit_cast(uint32_t, o);
}
__device__ __forceinline__ uint32_t codes4(uint32_t lo, uint32_t hi, float scale, _Float16) {
  i16x2 o = {0, 0};
  o = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(o, __builtin_bit_cast(f16x2, lo), scale, false);
  o = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(o, __builtin_bit_cast(f16x2, hi), scale, true);
  return __builtin_bit_cast(uint32_t, o);
}
__device__ __forceinline__ uint32_t codes4(uint32_t a, uint32_t b, uint32_t c, uint32_t d, float scale) {
  i16x2 o = {0, 0};
  o = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(o, __uint_as_float(a), __uint_as_float(b), scale, false);
  o = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(o, __uint_as_float(c), __uint_as_float(d), scale, true);
  return __builtin_bit_cast(uint32_t, o);
}

// A thread's 8 x 8 values and what a quantization asks of them.
template <typename T>
struct Square {  // 16-bit
  using P = Pair<T>;
  static constexpr int kRowMost = 4, kColMost = 4;  // words of maxima: two rows, two columns each
  uint32_t w[8][4];
  __device__ __forceinline__ void load(int i, const T* at) {
    const u32x4 v = *reinterpret_cast<const u32x4_any*>(at);
#pragma unroll
    for (int k = 0; k < 4; ++k) w[i][k] = v[k];
  }
  __device__ __forceinline__ void load(int i, const T* at, int64_t left) {
    const uint16_t* u = reinterpret_cast<const uint16_t*>(at);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t lo = 2 * k < left ? u[2 * k] : 0, hi = 2 * k + 1 < left ? u[2 * k + 1] : 0;
      w[i][k] = lo | hi << 16;
    }
  }
  __device__ __forceinline__ static uint32_t larger(uint32_t a, uint32_t b) { return P::larger(a, b); }
  __device__ __forceinline__ void maxima(uint32_t (&row)[4], uint32_t (&col)[4]) const {
    uint32_t one[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) col[k] = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t m[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        m[k] = w[i][k] & 0x7FFF7FFFu;
        col[k] = larger(col[k], m[k]);
      }
      one[i] = larger(larger(m[0], m[1]), larger(m[2], m[3]));
    }
    // Two rows a word: the larger of each row's even and odd columns.
#pragma unroll
    for (int i = 0; i < 4; ++i)
      row[i] = larger(__builtin_amdgcn_perm(one[2 * i + 1], one[2 * i], 0x05040100u),
                      __builtin_amdgcn_perm(one[2 * i + 1], one[2 * i], 0x07060302u));
  }
  __device__ __forceinline__ static bool odd(uint32_t m) {  // not finite
    return (m & 0xFFFFu) >= P::inf || (m >> 16) >= P::inf;
  }
  // The float32 bits of maximum i of the words.
  __device__ __forceinline__ static uint32_t bits(const uint32_t (&m)[4], int i) {
    return P::bits(i & 1 ? m[i >> 1] >> 16 : m[i >> 1] & 0xFFFFu);
  }
  // The maxima of the finite values.
  __device__ __forceinline__ void finite_maxima(uint32_t (&row)[4], uint32_t (&col)[4]) const {
    Square kept;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t lo = w[i][k] & 0x7FFFu, hi = w[i][k] & 0x7FFF0000u;
        kept.w[i][k] = (lo < P::inf ? lo : 0u) | (hi < P::inf << 16 ? hi : 0u);
      }
    kept.maxima(row, col);
  }
  __device__ __forceinline__ u32x2 row_codes(int i, float scale) const {
    return u32x2{codes4(w[i][0], w[i][1], scale, T{}), codes4(w[i][2], w[i][3], scale, T{})};
  }
  __device__ __forceinline__ u32x2 col_codes(int k, float scale) const {
    uint32_t p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      p[i] = __builtin_amdgcn_perm(w[2 * i + 1][k >> 1], w[2 * i][k >> 1], k & 1 ? 0x07060302u : 0x05040100u);
    return u32x2{codes4(p[0], p[1], scale, T{}), codes4(p[2], p[3], scale, T{})};
  }
  __device__ __forceinline__ float value(int i, int k) const { return P{w[i][k >> 1]}.value(k & 1); }
};

template <>
struct Square<float> {
  static constexpr int kRowMost = 8, kColMost = 8;
  static constexpr uint32_t inf = 0x7F800000u;
  uint32_t w[8][8];
  __device__ __forceinline__ void load(int i, const float* at) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const u32x4 v = *reinterpret_cast<const u32x4_any*>(at + 4 * h);
#pragma unroll
      for (int k = 0; k < 4; ++k) w[i][4 * h + k] = v[k];
    }
  }
  __device__ __forceinline__ void load(int i, const float* at, int64_t left) {
#pragma unroll
    for (int k = 0; k < 8; ++k) w[i][k] = k < left ? __float_as_uint(at[k]) : 0;
  }
  __device__ __forceinline__ static uint32_t larger(uint32_t a, uint32_t b) { return max(a, b); }
  __device__ __forceinline__ void maxima(uint32_t (&row)[8], uint32_t (&col)[8]) const {
#pragma unroll
    for (int k = 0; k < 8; ++k) row[k] = col[k] = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t m = w[i][k] & 0x7FFFFFFFu;
        row[i] = max(row[i], m);
        col[k] = max(col[k], m);
      }
  }
  __device__ __forceinline__ static bool odd(uint32_t m) { return m >= inf; }
  __device__ __forceinline__ static uint32_t bits(const uint32_t (&m)[8], int i) { return m[i]; }
  __device__ __forceinline__ void finite_maxima(uint32_t (&row)[8], uint32_t (&col)[8]) const {
#pragma unroll
    for (int k = 0; k < 8; ++k) row[k] = col[k] = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t b = w[i][k] & 0x7FFFFFFFu, m = b < inf ? b : 0u;
        row[i] = max(row[i], m);
        col[k] = max(col[k], m);
      }
  }
  __device__ __forceinline__ u32x2 row_codes(int i, float scale) const {
    return u32x2{codes4(w[i][0], w[i][1], w[i][2], w[i][3], scale),
                 codes4(w[i][4], w[i][5], w[i][6], w[i][7], scale)};
  }
  __device__ __forceinline__ u32x2 col_codes(int k, float scale) const {
    return u32x2{codes4(w[0][k], w[1][k], w[2][k], w[3][k], scale),
                 codes4(w[4][k], w[5][k], w[6][k], w[7][k], scale)};
  }
  __device__ __forceinline__ float value(int i, int k) const { return __uint_as_float(w[i][k]); }
};

// The largest over a row of 16 lanes.
template <int N>
__device__ __forceinline__ uint32_t turned_row(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x120 | N, 0xF, 0xF, false);  // row_ror:N
}

}  // namespace dionw

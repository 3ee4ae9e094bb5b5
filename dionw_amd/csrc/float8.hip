// 8-bit floating-point matrices with a scale for each block of 128, their products, and the
// quantization that makes them.
//
// A quantized matrix holds e4m3 codes (4 exponent bits, bias 7, 3 fraction bits, largest 448)
// row-major, its columns padded with zeros to a multiple of 128, and for every row and block
// of 128 columns the exponent byte of a float32 power of two. The powers are the smallest
// that bring the block's largest magnitude to 448 at most: they scale without rounding, cost
// no fraction bit, and instructions multiply by them on the way, so that a product is one
// accumulation in float32 from the first block to the last. Bytes are kept by column block,
// [blocks][rows], so that the rows of a tile lie side by side.
//
// Products run on one of two instructions, by their output's type:
// - float16 and bfloat16: v_mfma_scale_f32_16x16x128_f8f6f4, one block deep, scales
//   included, at twice the 16-bit rate. It adds groups of 8 products after cutting each to
//   13 bits below the exponent of the group's largest (measured: beside 2^16, 2^3 counts and
//   2^2 does not), and adds the groups in float32. On normal random operands the result is
//   1.3e-5 off (2-norm), on log-normal ones 6e-5: below the output's rounding (2e-4, 2e-3).
// - float32: v_mfma_f32_16x16x32_bf16 on codes expanded to bfloat16, scale included, which is
//   exact: 3e-8 off, the accumulation's own rounding. Weight gradients and whatever else asks
//   for float32 sums get them.
//
// A weight's bytes are equal within each 128 x 128 tile, so that its transpose holds the
// same values; an activation's differ from row to row.
#include "common.h"

#include <algorithm>
#include <mutex>

namespace dionw {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

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

// ---- quantization ------------------------------------------------------------------
//
// A workgroup takes a 128 x 128 tile: thread t the rows 8 (t / 16) .. + 7 and the columns
// 8 (t % 16) .. + 7, read once and held in registers. From them come the codes by rows and,
// through LDS, the codes of the transpose, each in whole 128-byte lines.
// Bound: HBM, 2 or 4 bytes read and 1 or 2 written an element.
struct QuantizeArgs {
  const void* x;
  int64_t rows, cols, ld;
  uint8_t* data;      // [rows][data_ld] or null
  int64_t data_ld;
  uint8_t* scale;     // [blocks][scale_ld]
  int64_t scale_ld;
  uint8_t* data_t;    // the transpose: [cols][data_t_ld] or null
  int64_t data_t_ld;
  uint8_t* scale_t;
  int64_t scale_t_ld;
  float* sums;        // [row tiles][cols]: each tile's column sums, or null
  int32_t tiles_c;
  int32_t vec;        // rows start at multiples of 16 bytes
};

template <typename T, bool TILES>
__global__ __launch_bounds__(256) void float8_quantize_kernel(QuantizeArgs q) {
  constexpr int kPitch = kTile + 16;
  __shared__ __attribute__((aligned(16))) uint8_t turned[kTile * kPitch];
  __shared__ uint32_t col_most[4][kTile];
  __shared__ float col_sum[4][kTile];
  __shared__ uint8_t row_bytes[kTile], col_bytes[kTile];
  const int tid = threadIdx.x, wave = tid >> 6;
  const int64_t r0 = (int64_t)(blockIdx.x / q.tiles_c) * kTile;
  const int64_t c0 = (int64_t)(blockIdx.x % q.tiles_c) * kTile;
  const int tr = tid / 16 * 8, tc = tid % 16 * 8;  // the thread's first row and column
  float v[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t r = r0 + tr + i, c = c0 + tc;
    const T* at = reinterpret_cast<const T*>(q.x) + r * q.ld + c;
    if (r < q.rows && q.vec && c + 8 <= q.cols) {
      T raw[8];
#pragma unroll
      for (int k = 0; k < (int)sizeof(T) / 2; ++k)
        reinterpret_cast<u32x4*>(raw)[k] = reinterpret_cast<const u32x4*>(at)[k];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[i][k] = to_float(raw[k]);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[i][k] = r < q.rows && c + k < q.cols ? to_float(at[k]) : 0.f;
    }
  }
  uint32_t row_most[8], most[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) row_most[i] = most[i] = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t b = magnitude(v[i][k]);
      row_most[i] = max(row_most[i], b);
      most[k] = max(most[k], b);
    }
#pragma unroll
  for (int off = 8; off >= 1; off >>= 1)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      row_most[i] = max(row_most[i], (uint32_t)__shfl_xor((int)row_most[i], off, kWave));
  if (TILES || q.data_t) {
#pragma unroll
    for (int off = 32; off >= 16; off >>= 1)
#pragma unroll
      for (int k = 0; k < 8; ++k)
        most[k] = max(most[k], (uint32_t)__shfl_xor((int)most[k], off, kWave));
    if ((tid & 63) < 16)
#pragma unroll
      for (int k = 0; k < 8; ++k) col_most[wave][tc + k] = most[k];
  }
  if (q.sums) {
    float s[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      s[k] = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) s[k] += v[i][k];
    }
#pragma unroll
    for (int off = 16; off <= 32; off <<= 1)
#pragma unroll
      for (int k = 0; k < 8; ++k) s[k] += __shfl_xor(s[k], off, kWave);
    if ((tid & 63) < 16)
#pragma unroll
      for (int k = 0; k < 8; ++k) col_sum[wave][tc + k] = s[k];
  }
  uint32_t row_byte[8], col_byte[8];
  if (TILES || q.data_t || q.sums) __syncthreads();
  if (TILES || q.data_t) {
    uint32_t all = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      uint32_t m = 0;
#pragma unroll
      for (int w = 0; w < 4; ++w) m = max(m, col_most[w][tc + k]);
      col_byte[k] = scale_byte(m);
      all = max(all, m);
    }
    if (TILES) {
#pragma unroll
      for (int off = 8; off >= 1; off >>= 1) all = max(all, (uint32_t)__shfl_xor((int)all, off, kWave));
#pragma unroll
      for (int k = 0; k < 8; ++k) col_byte[k] = row_byte[k] = scale_byte(all);
    }
  }
  if (!TILES)
#pragma unroll
    for (int i = 0; i < 8; ++i) row_byte[i] = scale_byte(row_most[i]);
  if (q.sums && tid < kTile && c0 + tid < q.cols)
    q.sums[r0 / kTile * q.cols + c0 + tid] =
        (col_sum[0][tid] + col_sum[1][tid]) + (col_sum[2][tid] + col_sum[3][tid]);
  if (q.data) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float inv = power(254 - row_byte[i]);
      u32x2 w;
      w[0] = pack4(v[i][0], v[i][1], v[i][2], v[i][3], inv);
      w[1] = pack4(v[i][4], v[i][5], v[i][6], v[i][7], inv);
      if (r0 + tr + i < q.rows)
        *reinterpret_cast<u32x2*>(q.data + (r0 + tr + i) * q.data_ld + c0 + tc) = w;
      if (tid % 16 == 0) row_bytes[tr + i] = (uint8_t)row_byte[i];
    }
  }
  if (q.data_t) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float inv = power(254 - col_byte[k]);
      u32x2 w;
      w[0] = pack4(v[0][k], v[1][k], v[2][k], v[3][k], inv);
      w[1] = pack4(v[4][k], v[5][k], v[6][k], v[7][k], inv);
      *reinterpret_cast<u32x2*>(turned + (tc + k) * kPitch + tr) = w;
    }
    if (tid < 16)
#pragma unroll
      for (int k = 0; k < 8; ++k) col_bytes[tc + k] = (uint8_t)col_byte[k];
  }
  __syncthreads();
  if (q.data && tid < kTile && r0 + tid < q.scale_ld)
    q.scale[c0 / kTile * q.scale_ld + r0 + tid] = row_bytes[tid];
  if (q.data_t) {
    if (tid < kTile && c0 + tid < q.scale_t_ld)
      q.scale_t[r0 / kTile * q.scale_t_ld + c0 + tid] = col_bytes[tid];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = j * 32 + tid / 8, at = tid % 8 * 16;
      if (c0 + c < q.cols)
        *reinterpret_cast<u32x4*>(q.data_t + (c0 + c) * q.data_t_ld + r0 + at) =
            *reinterpret_cast<const u32x4*>(turned + c * kPitch + at);
    }
  }
}

// out[c] = the parts' sums in order.
template <typename T>
__global__ __launch_bounds__(256) void sum_parts_kernel(const float* parts, int64_t count,
                                                        int64_t cols, T* out) {
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= cols) return;
  float s = 0.f;
  for (int64_t i = 0; i < count; ++i) s += parts[i * cols + c];
  out[c] = (T)s;
}

template <typename T>
int launch_quantize(const QuantizeArgs& q, bool tiles, unsigned grid, hipStream_t stream) {
  if (tiles)
    hipLaunchKernelGGL((float8_quantize_kernel<T, true>), dim3(grid), dim3(256), 0, stream, q);
  else
    hipLaunchKernelGGL((float8_quantize_kernel<T, false>), dim3(grid), dim3(256), 0, stream, q);
  return check_launch("float8_quantize");
}

// ---- products ------------------------------------------------------------------------

struct ProductArgs {
  const uint8_t* a;
  int64_t lda;
  const uint8_t* a_scale;
  int64_t a_scale_ld;
  const uint8_t* b;
  int64_t ldb;
  const uint8_t* b_scale;
  int64_t b_scale_ld;
  const float* bias;
  void* c;
  int64_t ldc;
  int64_t m, n;
  int32_t blocks;  // of 128 columns
  int32_t tiles_n;
};

// The scaled product of a fragment: 16 rows of each operand over one block. Either operand's
// lane i holds row i % 16 and the 32 bytes of its place i / 16 in the block; any order of the
// block's bytes serves that both share. D: lane i holds rows 4 (i / 16) .. + 3 of the first
// operand against row i % 16 of the second.
__device__ __forceinline__ f32x4 mfma(i32x8 a, i32x8 b, f32x4 c, int a_byte, int b_byte) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, a_byte, 0, b_byte);
}

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// Eight codes and their scale as bfloat16, exactly (a code has 4 significant bits).
__device__ __forceinline__ bf16x8 expand(int lo, int hi, float scale) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
  return __builtin_shufflevector(__builtin_shufflevector(a, b, 0, 1, 2, 3),
                                 __builtin_shufflevector(c, d, 0, 1, 2, 3), 0, 1, 2, 3, 4, 5, 6, 7);
}

// The scale that a row's codes are expanded with: half of theirs, as 448 x 2^120 (what a
// block of magnitudes up to the largest float32 may round to) is past bfloat16. Sums take
// kExpanded back in the epilogue.
__device__ __forceinline__ float half_power(int byte) { return __uint_as_float((uint32_t)(byte - 1) << 23); }
constexpr float kExpanded = 4.f;

// The same product summed in float32 throughout, in units of 1 / kExpanded.
__device__ __forceinline__ f32x4 mfma_exact(i32x8 a, i32x8 b, f32x4 c, float a_scale, float b_scale) {
#pragma unroll
  for (int q = 0; q < 4; ++q)
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(expand(a[2 * q], a[2 * q + 1], a_scale),
                                                expand(b[2 * q], b[2 * q + 1], b_scale), c, 0, 0, 0);
  return c;
}

// 64 x 64 outputs of 4 waves, 32 x 32 each, fragments read from memory.
template <typename OUT>
__global__ __launch_bounds__(256) void float8_gemm_kernel(ProductArgs g) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t m0 = (int64_t)(blockIdx.x / g.tiles_n) * 64 + (wave >> 1) * 32;
  const int64_t n0 = (int64_t)(blockIdx.x % g.tiles_n) * 64 + (wave & 1) * 32;
  const int i16 = lane & 15, G = lane >> 4;
  f32x4 acc[2][2] = {};
  int64_t row[2], col[2];
  for (int f = 0; f < 2; ++f) {
    row[f] = min(m0 + f * 16 + i16, g.m - 1);
    col[f] = min(n0 + f * 16 + i16, g.n - 1);
  }
  for (int kb = 0; kb < g.blocks; ++kb) {
    i32x8 a[2], b[2];
    int as[2], bs[2];
    for (int f = 0; f < 2; ++f) {
      const i32x4* pa = reinterpret_cast<const i32x4*>(g.a + row[f] * g.lda + kb * kTile + 32 * G);
      const i32x4* pb = reinterpret_cast<const i32x4*>(g.b + col[f] * g.ldb + kb * kTile + 32 * G);
      a[f] = __builtin_shufflevector(pa[0], pa[1], 0, 1, 2, 3, 4, 5, 6, 7);
      b[f] = __builtin_shufflevector(pb[0], pb[1], 0, 1, 2, 3, 4, 5, 6, 7);
      as[f] = g.a_scale[kb * g.a_scale_ld + row[f]];
      bs[f] = g.b_scale[kb * g.b_scale_ld + col[f]];
    }
    for (int i = 0; i < 2; ++i)
      for (int j = 0; j < 2; ++j)
        acc[i][j] = sizeof(OUT) == 4
                        ? mfma_exact(b[j], a[i], acc[i][j], half_power(bs[j]), half_power(as[i]))
                        : mfma(b[j], a[i], acc[i][j], bs[j], as[i]);
  }
  OUT* c = reinterpret_cast<OUT*>(g.c);
  for (int i = 0; i < 2; ++i)
    for (int j = 0; j < 2; ++j)
      for (int e = 0; e < 4; ++e) {
        const int64_t r = m0 + i * 16 + i16, q = n0 + j * 16 + 4 * G + e;
        if (r < g.m && q < g.n) 
          c[r * g.ldc + q] = (OUT)((sizeof(OUT) == 4 ? kExpanded : 1.f) * acc[i][j][e] + (g.bias ? g.bias[q] : 0.f));
      }
}

template <typename OUT>
int launch_product(ProductArgs g, hipStream_t stream) {
  const int64_t tm = ceil_div(g.m, 64), tn = ceil_div(g.n, 64);
  DIONW_REQUIRE(tm * tn < INT32_MAX, "float8_gemm: too many tiles");
  g.tiles_n = (int32_t)tn;
  hipLaunchKernelGGL(float8_gemm_kernel<OUT>, dim3((unsigned)(tm * tn)), dim3(256), 0, stream, g);
  return check_launch("float8_gemm");
}

}  // namespace
}  // namespace dionw

using namespace dionw;

extern "C" {

int dionw_float8_quantize(int32_t elem, const void* x, int64_t rows, int64_t cols, int64_t ld,
                          int32_t tiles, void* data, int64_t data_ld, void* scale,
                          int64_t scale_ld, void* data_t, int64_t data_t_ld, void* scale_t,
                          int64_t scale_t_ld, float* sums, hipStream_t stream) {
  DIONW_REQUIRE(elem == kF16 || elem == kBF16 || elem == kF32, "float8_quantize: bad element type %d", elem);
  DIONW_REQUIRE(rows >= 0 && cols >= 0, "float8_quantize: negative extent");
  if (rows == 0 || cols == 0) return kOk;
  DIONW_REQUIRE(data || data_t || sums, "float8_quantize: no output");
  DIONW_REQUIRE(x && ld >= cols, "float8_quantize: bad input");
  auto fits = [](const void* d, int64_t d_ld, const void* s, int64_t s_ld, int64_t r, int64_t c) {
    return !d || (s && d_ld >= round_up(c, kTile) && d_ld % 16 == 0 && s_ld >= r && aligned16(d));
  };
  DIONW_REQUIRE(fits(data, data_ld, scale, scale_ld, rows, cols) &&
                    fits(data_t, data_t_ld, scale_t, scale_t_ld, cols, rows),
                "float8_quantize: an output is too small or not aligned");
  const int64_t tr = ceil_div(rows, kTile), tc = ceil_div(cols, kTile);
  DIONW_REQUIRE(tr < INT32_MAX / tc, "float8_quantize: too many tiles");
  const int64_t size = elem == kF32 ? 4 : 2;
  QuantizeArgs q{x,       rows,     cols,    ld,
                 static_cast<uint8_t*>(data),   data_ld,   static_cast<uint8_t*>(scale),   scale_ld,
                 static_cast<uint8_t*>(data_t), data_t_ld, static_cast<uint8_t*>(scale_t), scale_t_ld,
                 sums,    (int32_t)tc,
                 aligned16(x) && ld * size % 16 == 0};
  const unsigned grid = (unsigned)(tr * tc);
  if (elem == kF16) return launch_quantize<_Float16>(q, tiles != 0, grid, stream);
  if (elem == kBF16) return launch_quantize<__bf16>(q, tiles != 0, grid, stream);
  return launch_quantize<float>(q, tiles != 0, grid, stream);
}

int dionw_sum_parts(const float* parts, int64_t count, int64_t cols, int32_t elem, void* out,
                    hipStream_t stream) {
  DIONW_REQUIRE(count >= 0 && cols >= 0, "sum_parts: negative extent");
  if (cols == 0) return kOk;
  DIONW_REQUIRE(out && (parts || count == 0), "sum_parts: null pointer");
  DIONW_REQUIRE(ceil_div(cols, 256) < INT32_MAX, "sum_parts: too many columns");
  const dim3 grid((unsigned)ceil_div(cols, 256));
  if (elem == kF16)
    hipLaunchKernelGGL(sum_parts_kernel<_Float16>, grid, dim3(256), 0, stream, parts, count, cols,
                       static_cast<_Float16*>(out));
  else if (elem == kBF16)
    hipLaunchKernelGGL(sum_parts_kernel<__bf16>, grid, dim3(256), 0, stream, parts, count, cols,
                       static_cast<__bf16*>(out));
  else if (elem == kF32)
    hipLaunchKernelGGL(sum_parts_kernel<float>, grid, dim3(256), 0, stream, parts, count, cols,
                       static_cast<float*>(out));
  else
    DIONW_REQUIRE(false, "sum_parts: bad element type %d", elem);
  return check_launch("sum_parts");
}

int dionw_float8_gemm(int64_t m, int64_t n, int64_t depth, const void* a, int64_t lda,
                      const void* a_scale, int64_t a_scale_ld, const void* b, int64_t ldb,
                      const void* b_scale, int64_t b_scale_ld, const float* bias, int32_t elem,
                      void* c, int64_t ldc, hipStream_t stream) {
  DIONW_REQUIRE(m >= 0 && n >= 0 && depth >= 0 && depth % kTile == 0,
                "float8_gemm: bad extents %lld x %lld x %lld", (long long)m, (long long)n,
                (long long)depth);
  DIONW_REQUIRE(elem == kF16 || elem == kBF16 || elem == kF32, "float8_gemm: bad element type %d", elem);
  if (m == 0 || n == 0) return kOk;
  DIONW_REQUIRE(c && ldc >= n, "float8_gemm: bad output");
  DIONW_REQUIRE(depth == 0 || (a && a_scale && b && b_scale), "float8_gemm: null operand");
  DIONW_REQUIRE(depth / kTile < INT32_MAX, "float8_gemm: depth too large");
  DIONW_REQUIRE(lda >= depth && ldb >= depth && lda % 16 == 0 && ldb % 16 == 0 && aligned16(a) &&
                    aligned16(b) && a_scale_ld >= m && b_scale_ld >= n,
                "float8_gemm: operands need rows of at least their depth at multiples of 16 bytes "
                "and a scale for each row");
  ProductArgs g{static_cast<const uint8_t*>(a), lda, static_cast<const uint8_t*>(a_scale), a_scale_ld,
                static_cast<const uint8_t*>(b), ldb, static_cast<const uint8_t*>(b_scale), b_scale_ld,
                bias, c, ldc, m, n, (int32_t)(depth / kTile), 0};
  if (elem == kF16) return launch_product<_Float16>(g, stream);
  if (elem == kBF16) return launch_product<__bf16>(g, stream);
  return launch_product<float>(g, stream);
}

}  // extern "C"

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
// A weight's bytes are equal within each 128 x 128 tile, so that its transpose holds the
// same values; an activation's differ from row to row.
#include "float8.h"

namespace dionw {
namespace {

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
  uint8_t* data_t;    // the transpose: [cols][data_t_ld bytes] or null
  int64_t data_t_ld;
  uint8_t* scale_t;
  int64_t scale_t_ld;
  float* sums;        // [row tiles][cols]: each tile's column sums, or null
  int32_t tiles_c;
  int32_t vec;        // rows start at multiples of 16 bytes
  int32_t expand_t;   // the transpose in bfloat16, scales included
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
  if (q.data_t && q.expand_t) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = j * 32 + tid / 8, at = tid % 8 * 16;
      if (c0 + c >= q.cols) continue;
      const u32x4 w = *reinterpret_cast<const u32x4*>(turned + c * kPitch + at);
      const float scale = half_power(col_bytes[c]);
      bf16x8* out = reinterpret_cast<bf16x8*>(q.data_t + (c0 + c) * q.data_t_ld + 2 * (r0 + at));
      out[0] = expand(w[0], w[1], scale);
      out[1] = expand(w[2], w[3], scale);
    }
  } else if (q.data_t) {
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

// Codes to bfloat16 halves of their values, 16 a thread.
__global__ __launch_bounds__(256) void float8_expand_kernel(const uint8_t* data, int64_t data_ld,
                                                            const uint8_t* scale, int64_t scale_ld,
                                                            int64_t rows, int64_t chunks,
                                                            __bf16* out, int64_t out_ld) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = at / chunks, c = (at - row * chunks) * 16;
  if (row >= rows) return;
  const u32x4 w = *reinterpret_cast<const u32x4*>(data + row * data_ld + c);
  const float s = half_power(scale[c / kTile * scale_ld + row]);
  bf16x8* to = reinterpret_cast<bf16x8*>(out + row * out_ld + c);
  to[0] = expand(w[0], w[1], s);
  to[1] = expand(w[2], w[3], s);
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

}  // namespace
}  // namespace dionw

using namespace dionw;

extern "C" {

int dionw_float8_quantize(int32_t elem, const void* x, int64_t rows, int64_t cols, int64_t ld,
                          int32_t tiles, void* data, int64_t data_ld, void* scale,
                          int64_t scale_ld, void* data_t, int64_t data_t_ld, void* scale_t,
                          int64_t scale_t_ld, int32_t expand_t, float* sums, hipStream_t stream) {
  DIONW_REQUIRE(elem == kF16 || elem == kBF16 || elem == kF32, "float8_quantize: bad element type %d", elem);
  DIONW_REQUIRE(rows >= 0 && cols >= 0, "float8_quantize: negative extent");
  if (rows == 0 || cols == 0) return kOk;
  DIONW_REQUIRE(data || data_t || sums, "float8_quantize: no output");
  DIONW_REQUIRE(x && ld >= cols, "float8_quantize: bad input");
  auto fits = [](const void* d, int64_t d_ld, const void* s, int64_t s_ld, int64_t r, int64_t c) {
    return !d || (s && d_ld >= round_up(c, kTile) && d_ld % 16 == 0 && s_ld >= r && aligned16(d));
  };
  DIONW_REQUIRE(fits(data, data_ld, scale, scale_ld, rows, cols) &&
                    fits(data_t, data_t_ld, expand_t ? x : scale_t, expand_t ? cols : scale_t_ld, cols, rows),
                "float8_quantize: an output is too small or not aligned");
  const int64_t tr = ceil_div(rows, kTile), tc = ceil_div(cols, kTile);
  DIONW_REQUIRE(tr < INT32_MAX / tc, "float8_quantize: too many tiles");
  const int64_t size = elem == kF32 ? 4 : 2;
  QuantizeArgs q{x,       rows,     cols,    ld,
                 static_cast<uint8_t*>(data),   data_ld,   static_cast<uint8_t*>(scale),   scale_ld,
                 static_cast<uint8_t*>(data_t), expand_t ? 2 * data_t_ld : data_t_ld,
                 static_cast<uint8_t*>(scale_t), scale_t_ld,
                 sums,    (int32_t)tc,
                 aligned16(x) && ld * size % 16 == 0, expand_t};
  const unsigned grid = (unsigned)(tr * tc);
  if (elem == kF16) return launch_quantize<_Float16>(q, tiles != 0, grid, stream);
  if (elem == kBF16) return launch_quantize<__bf16>(q, tiles != 0, grid, stream);
  return launch_quantize<float>(q, tiles != 0, grid, stream);
}

int dionw_float8_expand(const void* data, int64_t data_ld, const void* scale, int64_t scale_ld,
                        int64_t rows, int64_t depth, void* out, int64_t out_ld,
                        hipStream_t stream) {
  DIONW_REQUIRE(rows >= 0 && depth >= 0 && depth % kTile == 0, "float8_expand: bad extents");
  if (rows == 0 || depth == 0) return kOk;
  DIONW_REQUIRE(data && scale && out && aligned16(data) && aligned16(out) && data_ld >= depth &&
                    data_ld % 16 == 0 && out_ld >= depth && out_ld % 8 == 0 && scale_ld >= rows,
                "float8_expand: a matrix is too small or not aligned");
  const int64_t chunks = depth / 16;
  DIONW_REQUIRE(rows <= (int64_t)INT32_MAX * 256 / chunks, "float8_expand: too many elements");
  hipLaunchKernelGGL(float8_expand_kernel, dim3((unsigned)ceil_div(rows * chunks, 256)), dim3(256), 0,
                     stream, static_cast<const uint8_t*>(data), data_ld,
                     static_cast<const uint8_t*>(scale), scale_ld, rows, chunks,
                     static_cast<__bf16*>(out), out_ld);
  return check_launch("float8_expand");
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

}  // extern "C"

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

// The most workgroups of 256 a launch takes (2^32 threads).
constexpr int64_t kMostGroups = (int64_t{1} << 24) - 1;

// ---- quantization ------------------------------------------------------------------
//
// A workgroup takes a 128 x 128 tile: thread t the rows 8 (t / 16) .. + 7 and the columns
// 8 (t % 16) .. + 7, read once and held as they are. From them come the codes by rows and,
// through LDS, the codes of the transpose, each in whole 128-byte lines. Magnitudes are compared
// as integers (16-bit ones two at a time), and v_cvt_scalef32_pk_fp8_* rounds two values a time,
// scale included. Infinities and NaN become NaN codes by themselves; a thread whose maximum is one
// of them takes its finite values' maxima on a path of its own.
// Bound: HBM, 2 or 4 bytes read and 1 to 4 written an element. 8192 x 4096 bfloat16 both ways 28 us
// (4.8 TB/s), 8192 x 14336 with the transpose expanded 115 us (5.1), a 14336 x 4096 float32 weight by
// tiles both ways 68 us (5.2); with every value converted to float32 first 43, 211 and 69 us.
struct Output {
  uint8_t* data;     // null: not asked for
  int64_t ld;        // bytes
  uint8_t* scale;    // codes only
  int64_t scale_ld;
  int32_t expanded;  // bfloat16 halves of the values instead of codes
};
struct QuantizeArgs {
  const void* x;
  int64_t rows, cols, ld;
  Output by_row, by_col;  // x, and its transpose
  float* sums;            // [row tiles][cols]: each tile's column sums, or null
  int32_t tiles_c;
};

// A thread's 8 x 8 values and what the kernel asks of them.
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

// Eight values of a row, and the float32 bits of their largest finite magnitude.
template <typename T>
struct Line {
  Square<T> s;  // its first row
  __device__ __forceinline__ void load(const T* at) { s.load(0, at); }
  __device__ __forceinline__ void load(const T* at, int64_t left) { s.load(0, at, left); }
  __device__ __forceinline__ uint32_t most() const {
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t b = __float_as_uint(s.value(0, k)) & 0x7FFFFFFFu;
      m = max(m, b < 0x7F800000u ? b : 0u);
    }
    return m;
  }
  __device__ __forceinline__ u32x2 codes(float scale) const { return s.row_codes(0, scale); }
};

// A workgroup's LDS.
struct Shared {
  // Bytes of the transpose: 33 words a row, so that the 16 columns x 4 row groups of a wave's
  // 8-byte writes spread over the banks.
  static constexpr int pitch = 33;
  uint32_t turned[kTile * pitch];
  uint32_t col_most[4][16][8];
  float col_sum[4][kTile];
  uint8_t row_bytes[kTile], col_bytes[kTile];
};

template <typename T, bool TILES>
__device__ __forceinline__ void quantize_tile(const QuantizeArgs& q, uint32_t tile, Shared& shared) {
  using S = Square<T>;
  constexpr int RM = S::kRowMost, CM = S::kColMost, kPitch = Shared::pitch;
  auto& turned = shared.turned;
  auto& col_most = shared.col_most;
  auto& col_sum = shared.col_sum;
  auto& row_bytes = shared.row_bytes;
  auto& col_bytes = shared.col_bytes;
  const int tid = threadIdx.x, wave = tid >> 6;
  const int64_t r0 = (int64_t)(tile / q.tiles_c) * kTile;
  const int64_t c0 = (int64_t)(tile % q.tiles_c) * kTile;
  const int tr = tid / 16 * 8, tc = tid % 16 * 8;  // the thread's first row and column
  S v;
  const T* at = reinterpret_cast<const T*>(q.x) + (r0 + tr) * q.ld + c0 + tc;
  if (r0 + tr + 8 <= q.rows && c0 + tc + 8 <= q.cols) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v.load(i, at + i * q.ld);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      v.load(i, at + i * q.ld, r0 + tr + i < q.rows ? q.cols - c0 - tc : 0);
  }
  uint32_t row[RM], col[CM];
  v.maxima(row, col);
  uint32_t all = 0;
#pragma unroll
  for (int k = 0; k < CM; ++k) all = S::larger(all, col[k]);
  if (S::odd(all)) v.finite_maxima(row, col);
  if (!TILES) {
#pragma unroll
    for (int i = 0; i < RM; ++i) {
      row[i] = S::larger(row[i], turned_row<8>(row[i]));
      row[i] = S::larger(row[i], turned_row<4>(row[i]));
      row[i] = S::larger(row[i], turned_row<2>(row[i]));
      row[i] = S::larger(row[i], turned_row<1>(row[i]));
    }
  }
  if (TILES || q.by_col.data) {
#pragma unroll
    for (int k = 0; k < CM; ++k) {
      col[k] = S::larger(col[k], (uint32_t)__shfl_xor((int)col[k], 16, kWave));
      col[k] = S::larger(col[k], (uint32_t)__shfl_xor((int)col[k], 32, kWave));
    }
    if ((tid & 63) < 16)
#pragma unroll
      for (int k = 0; k < CM; ++k) col_most[wave][tid & 15][k] = col[k];
  }
  if (q.sums) {
    float s[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      s[k] = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) s[k] += v.value(i, k);
    }
#pragma unroll
    for (int off = 16; off <= 32; off <<= 1)
#pragma unroll
      for (int k = 0; k < 8; ++k) s[k] += __shfl_xor(s[k], off, kWave);
    if ((tid & 63) < 16)
#pragma unroll
      for (int k = 0; k < 8; ++k) col_sum[wave][tc + k] = s[k];
  }
  if (TILES || q.by_col.data || q.sums) __syncthreads();
  if (TILES || q.by_col.data) {
#pragma unroll
    for (int k = 0; k < CM; ++k)
      col[k] = S::larger(S::larger(col_most[0][tid & 15][k], col_most[1][tid & 15][k]),
                         S::larger(col_most[2][tid & 15][k], col_most[3][tid & 15][k]));
  }
  uint32_t tile_byte = 0;
  if (TILES) {
    uint32_t most = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) most = max(most, S::bits(col, k));
    most = max(most, turned_row<8>(most));
    most = max(most, turned_row<4>(most));
    most = max(most, turned_row<2>(most));
    most = max(most, turned_row<1>(most));
    tile_byte = scale_byte(most);
  }
  if (q.sums && tid < kTile && c0 + tid < q.cols)
    q.sums[r0 / kTile * q.cols + c0 + tid] =
        (col_sum[0][tid] + col_sum[1][tid]) + (col_sum[2][tid] + col_sum[3][tid]);
  if (q.by_row.data) {
    uint8_t* out = q.by_row.data + (r0 + tr) * q.by_row.ld;
#pragma unroll
    for (int i = 0; i < 8; ++i, out += q.by_row.ld) {
      const uint32_t byte = TILES ? tile_byte : scale_byte(S::bits(row, i));
      const u32x2 w = v.row_codes(i, power(byte));
      if (r0 + tr + i < q.rows) {
        if (q.by_row.expanded)
          *reinterpret_cast<bf16x8*>(out + 2 * (c0 + tc)) = expand(w[0], w[1], half_power(byte));
        else
          *reinterpret_cast<u32x2*>(out + c0 + tc) = w;
      }
      if (tid % 16 == 0) row_bytes[tr + i] = (uint8_t)byte;
    }
  }
  if (q.by_col.data) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t byte = TILES ? tile_byte : scale_byte(S::bits(col, k));
      const u32x2 w = v.col_codes(k, power(byte));
      turned[(tc + k) * kPitch + tr / 4] = w[0];
      turned[(tc + k) * kPitch + tr / 4 + 1] = w[1];
      if (tid < 16) col_bytes[tc + k] = (uint8_t)byte;
    }
  }
  __syncthreads();
  if (q.by_row.data && !q.by_row.expanded && tid < kTile && r0 + tid < q.by_row.scale_ld)
    q.by_row.scale[c0 / kTile * q.by_row.scale_ld + r0 + tid] = row_bytes[tid];
  if (!q.by_col.data) return;
  if (!q.by_col.expanded && tid < kTile && c0 + tid < q.by_col.scale_ld)
    q.by_col.scale[r0 / kTile * q.by_col.scale_ld + c0 + tid] = col_bytes[tid];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int c = j * 32 + tid / 8, word = tid % 8 * 4;
    if (c0 + c >= q.cols) continue;
    u32x4 w;
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = turned[c * kPitch + word + k];
    uint8_t* out = q.by_col.data + (c0 + c) * q.by_col.ld;
    if (q.by_col.expanded) {
      const float half = half_power(col_bytes[c]);
      bf16x8* to = reinterpret_cast<bf16x8*>(out + 2 * (r0 + 4 * word));
      to[0] = expand(w[0], w[1], half);
      to[1] = expand(w[2], w[3], half);
    } else {
      *reinterpret_cast<u32x4*>(out + r0 + 4 * word) = w;
    }
  }
}

template <typename T, bool TILES>
__global__ __launch_bounds__(256) void float8_quantize_kernel(QuantizeArgs q) {
  __shared__ Shared shared;
  quantize_tile<T, TILES>(q, blockIdx.x, shared);
}

// The same codes and scales by rows alone: 16 lanes take a row's block of 128, a workgroup 16
// rows' blocks, so that a matrix of a hundred rows still fills the GPU, and nothing goes through
// LDS. us in a chain of launches, here / on 128 x 128 tiles: float16 100 x 14336 4.2 / 6.2, 8192 x
// 4096 16.4 / 17.2; float32 64 x 4096 4.2 / 5.0, 8192 x 4096 23.9 / 25.8.
template <typename T>
__global__ __launch_bounds__(256) void float8_quantize_rows_kernel(QuantizeArgs q) {
  const int lane = threadIdx.x & 15;
  const int64_t row = (int64_t)(blockIdx.x / q.tiles_c) * 16 + threadIdx.x / 16;
  const int64_t block = blockIdx.x % q.tiles_c, c = block * kTile + 8 * lane;
  if (row >= q.rows) return;  // a row's 16 lanes together
  Line<T> v;
  const T* at = reinterpret_cast<const T*>(q.x) + row * q.ld + c;
  if (c + 8 <= q.cols) v.load(at);
  else v.load(at, q.cols - c);
  uint32_t most = v.most();
  most = max(most, turned_row<8>(most));
  most = max(most, turned_row<4>(most));
  most = max(most, turned_row<2>(most));
  most = max(most, turned_row<1>(most));
  const uint32_t byte = scale_byte(most);
  const u32x2 w = v.codes(power(byte));
  *reinterpret_cast<u32x2*>(q.by_row.data + row * q.by_row.ld + c) = w;
  if (lane == 0) q.by_row.scale[block * q.by_row.scale_ld + row] = (uint8_t)byte;
}

// Codes to bfloat16 halves of their values, 16 a thread.
struct ExpandArgs {
  const uint8_t* data;
  int64_t data_ld;
  const uint8_t* scale;
  int64_t scale_ld, rows, chunks;  // chunks: 16 codes each, of a row
  __bf16* out;
  int64_t out_ld;
};
__device__ __forceinline__ void expand_codes(const ExpandArgs& g, uint32_t block) {
  const int64_t at = (int64_t)block * 256 + threadIdx.x;
  const int64_t row = at / g.chunks, c = (at - row * g.chunks) * 16;
  if (row >= g.rows) return;
  const u32x4 w = *reinterpret_cast<const u32x4*>(g.data + row * g.data_ld + c);
  const float s = half_power(g.scale[c / kTile * g.scale_ld + row]);
  bf16x8* to = reinterpret_cast<bf16x8*>(g.out + row * g.out_ld + c);
  to[0] = expand(w[0], w[1], s);
  to[1] = expand(w[2], w[3], s);
}
__global__ __launch_bounds__(256) void float8_expand_kernel(ExpandArgs g) {
  expand_codes(g, blockIdx.x);
}

// What a linear layer's pass quantizes and expands, in one launch: a small layer's parts hide each
// other's latency.
template <typename TX, typename TW>
__global__ __launch_bounds__(256) void float8_quantize_pair_kernel(QuantizeArgs x, QuantizeArgs w,
                                                                   uint32_t x_tiles) {
  __shared__ Shared shared;
  if (blockIdx.x < x_tiles)
    quantize_tile<TX, false>(x, blockIdx.x, shared);
  else
    quantize_tile<TW, true>(w, blockIdx.x - x_tiles, shared);
}
template <typename T>
__global__ __launch_bounds__(256) void float8_quantize_expand_kernel(QuantizeArgs x, ExpandArgs a,
                                                                     ExpandArgs b, uint32_t x_tiles,
                                                                     uint32_t a_end) {
  __shared__ Shared shared;
  if (blockIdx.x < x_tiles)
    quantize_tile<T, false>(x, blockIdx.x, shared);
  else if (blockIdx.x < a_end)
    expand_codes(a, blockIdx.x - x_tiles);
  else
    expand_codes(b, blockIdx.x - a_end);
}

// out[c] = the parts' sums: 4 threads a column, a quarter of the parts each in order, then
// (0 + 1) + (2 + 3).
template <typename T>
__global__ __launch_bounds__(256) void sum_parts_kernel(const float* parts, int64_t count,
                                                        int64_t cols, T* out) {
  __shared__ float quarter[4][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t c = (int64_t)blockIdx.x * 64 + lane, per = (count + 3) / 4;
  const int64_t last = min(count, (w + 1) * per);
  float s = 0.f;
  if (c < cols)
#pragma unroll 8
    for (int64_t i = w * per; i < last; ++i) s += parts[i * cols + c];
  quarter[w][lane] = s;
  __syncthreads();
  if (w == 0 && c < cols)
    out[c] = (T)((quarter[0][lane] + quarter[1][lane]) + (quarter[2][lane] + quarter[3][lane]));
}

template <typename T>
int launch_quantize(const QuantizeArgs& q, bool tiles, unsigned grid, hipStream_t stream) {
  if (!tiles && !q.by_row.expanded && !q.by_col.data && !q.sums && ceil_div(q.rows, 16) * q.tiles_c <= kMostGroups) {
    hipLaunchKernelGGL(float8_quantize_rows_kernel<T>, dim3((unsigned)(ceil_div(q.rows, 16) * q.tiles_c)),
                       dim3(256), 0, stream, q);
    return check_launch("float8_quantize_rows");
  }
  if (tiles)
    hipLaunchKernelGGL((float8_quantize_kernel<T, true>), dim3(grid), dim3(256), 0, stream, q);
  else
    hipLaunchKernelGGL((float8_quantize_kernel<T, false>), dim3(grid), dim3(256), 0, stream, q);
  return check_launch("float8_quantize");
}

bool good_elem(int32_t e) { return e == kF16 || e == kBF16 || e == kF32; }

// Checks a quantization; `tiles`: its workgroups, 0 where there is nothing to do.
int prepare(const Quantization& j, QuantizeArgs& q, int64_t& tiles) {
  tiles = 0;
  DIONW_REQUIRE(good_elem(j.elem), "float8_quantize: bad element type %d", j.elem);
  DIONW_REQUIRE(j.rows >= 0 && j.cols >= 0, "float8_quantize: negative extent");
  if (j.rows == 0 || j.cols == 0) return kOk;
  DIONW_REQUIRE(j.by_row.data || j.by_col.data || j.sums, "float8_quantize: no output");
  DIONW_REQUIRE(j.x && j.ld >= j.cols, "float8_quantize: bad input");
  auto fits = [](const Matrix& o, bool expanded, int64_t r, int64_t c) {
    return !o.data || (o.depth >= round_up(c, kTile) && o.depth % 16 == 0 && aligned16(o.data) &&
                       (expanded || o.scale_ld >= r));
  };
  const bool row_expanded = !j.by_row.scale, col_expanded = !j.by_col.scale;
  DIONW_REQUIRE(fits(j.by_row, row_expanded, j.rows, j.cols) && fits(j.by_col, col_expanded, j.cols, j.rows),
                "float8_quantize: an output is too small or not aligned");
  const int64_t tr = ceil_div(j.rows, kTile), tc = ceil_div(j.cols, kTile);
  DIONW_REQUIRE(tr <= kMostGroups / tc, "float8_quantize: too many tiles");
  auto output = [](const Matrix& o, bool expanded) {
    return Output{static_cast<uint8_t*>(o.data), expanded ? 2 * o.depth : o.depth,
                  static_cast<uint8_t*>(o.scale), o.scale_ld, expanded};
  };
  q = {};
  q.x = j.x;
  q.rows = j.rows;
  q.cols = j.cols;
  q.ld = j.ld;
  q.by_row = output(j.by_row, row_expanded);
  q.by_col = output(j.by_col, col_expanded);
  q.sums = j.sums;
  q.tiles_c = (int32_t)tc;
  tiles = tr * tc;
  return kOk;
}

int prepare(const void* data, int64_t data_ld, const void* scale, int64_t scale_ld, int64_t rows,
            int64_t depth, void* out, int64_t out_ld, ExpandArgs& g, int64_t& blocks) {
  blocks = 0;
  DIONW_REQUIRE(rows >= 0 && depth >= 0 && depth % kTile == 0, "float8_expand: bad extents");
  if (rows == 0 || depth == 0) return kOk;
  DIONW_REQUIRE(data && scale && out && aligned16(data) && aligned16(out) && data_ld >= depth &&
                    data_ld % 16 == 0 && out_ld >= depth && out_ld % 8 == 0 && scale_ld >= rows,
                "float8_expand: a matrix is too small or not aligned");
  g = {static_cast<const uint8_t*>(data), data_ld, static_cast<const uint8_t*>(scale), scale_ld, rows,
       depth / 16, static_cast<__bf16*>(out), out_ld};
  DIONW_REQUIRE(rows <= kMostGroups * 256 / g.chunks, "float8_expand: too many elements");
  blocks = ceil_div(rows * g.chunks, 256);
  return kOk;
}

template <typename TX>
int launch_pair(const QuantizeArgs& x, int64_t x_tiles, int32_t w_elem, const QuantizeArgs& w,
                int64_t w_tiles, hipStream_t stream) {
  const dim3 grid((unsigned)(x_tiles + w_tiles));
  if (w_elem == kF16)
    hipLaunchKernelGGL((float8_quantize_pair_kernel<TX, _Float16>), grid, dim3(256), 0, stream, x, w,
                       (uint32_t)x_tiles);
  else if (w_elem == kBF16)
    hipLaunchKernelGGL((float8_quantize_pair_kernel<TX, __bf16>), grid, dim3(256), 0, stream, x, w,
                       (uint32_t)x_tiles);
  else
    hipLaunchKernelGGL((float8_quantize_pair_kernel<TX, float>), grid, dim3(256), 0, stream, x, w,
                       (uint32_t)x_tiles);
  return check_launch("float8_quantize_pair");
}

}  // namespace

int quantize_pair(const Quantization& x, const Quantization& w, hipStream_t stream) {
  QuantizeArgs qx{}, qw{};
  int64_t x_tiles, w_tiles;
  DIONW_TRY(prepare(x, qx, x_tiles));
  DIONW_TRY(prepare(w, qw, w_tiles));
  if (x_tiles + w_tiles == 0) return kOk;
  DIONW_REQUIRE(x_tiles + w_tiles <= kMostGroups, "float8_quantize: too many tiles");
  if (x.elem == kF16) return launch_pair<_Float16>(qx, x_tiles, w.elem, qw, w_tiles, stream);
  if (x.elem == kBF16) return launch_pair<__bf16>(qx, x_tiles, w.elem, qw, w_tiles, stream);
  return launch_pair<float>(qx, x_tiles, w.elem, qw, w_tiles, stream);
}

int quantize_and_expand(const Quantization& x, const Matrix (&from)[2], const Matrix (&to)[2],
                        hipStream_t stream) {
  QuantizeArgs q{};
  ExpandArgs g[2] = {};
  int64_t tiles = 0, blocks[2] = {0, 0};
  if (x.by_row.data || x.by_col.data || x.sums) DIONW_TRY(prepare(x, q, tiles));
  for (int i = 0; i < 2; ++i)
    if (to[i].data)
      DIONW_TRY(prepare(from[i].data, from[i].depth, from[i].scale, from[i].scale_ld, from[i].rows,
                        from[i].depth, to[i].data, to[i].depth, g[i], blocks[i]));
  const int64_t total = tiles + blocks[0] + blocks[1];
  if (total == 0) return kOk;
  DIONW_REQUIRE(total <= kMostGroups, "float8_quantize: too many tiles");
  auto launch = [&](auto kern) {
    hipLaunchKernelGGL(kern, dim3((unsigned)total), dim3(256), 0, stream, q, g[0], g[1], (uint32_t)tiles,
                       (uint32_t)(tiles + blocks[0]));
  };
  if (x.elem == kF16) launch(float8_quantize_expand_kernel<_Float16>);
  else if (x.elem == kBF16) launch(float8_quantize_expand_kernel<__bf16>);
  else launch(float8_quantize_expand_kernel<float>);
  return check_launch("float8_quantize_expand");
}

}  // namespace dionw

using namespace dionw;

extern "C" {

int dionw_float8_quantize(int32_t elem, const void* x, int64_t rows, int64_t cols, int64_t ld,
                          int32_t tiles, void* data, int64_t data_ld, void* scale,
                          int64_t scale_ld, void* data_t, int64_t data_t_ld, void* scale_t,
                          int64_t scale_t_ld, int32_t expanded, float* sums, hipStream_t stream) {
  const bool row_expanded = expanded & 1, col_expanded = expanded & 2;
  DIONW_REQUIRE((!data || row_expanded || scale) && (!data_t || col_expanded || scale_t),
                "float8_quantize: codes need their scales");
  const Quantization job{elem, x, rows, cols, ld,
                         {data, row_expanded ? nullptr : scale, rows, data_ld, scale_ld},
                         {data_t, col_expanded ? nullptr : scale_t, cols, data_t_ld, scale_t_ld}, sums};
  QuantizeArgs q{};
  int64_t count;
  DIONW_TRY(prepare(job, q, count));
  if (count == 0) return kOk;
  const unsigned grid = (unsigned)count;
  if (elem == kF16) return launch_quantize<_Float16>(q, tiles != 0, grid, stream);
  if (elem == kBF16) return launch_quantize<__bf16>(q, tiles != 0, grid, stream);
  return launch_quantize<float>(q, tiles != 0, grid, stream);
}

int dionw_float8_expand(const void* data, int64_t data_ld, const void* scale, int64_t scale_ld,
                        int64_t rows, int64_t depth, void* out, int64_t out_ld,
                        hipStream_t stream) {
  ExpandArgs g{};
  int64_t blocks;
  DIONW_TRY(prepare(data, data_ld, scale, scale_ld, rows, depth, out, out_ld, g, blocks));
  if (blocks == 0) return kOk;
  hipLaunchKernelGGL(float8_expand_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, g);
  return check_launch("float8_expand");
}

int dionw_sum_parts(const float* parts, int64_t count, int64_t cols, int32_t elem, void* out,
                    hipStream_t stream) {
  DIONW_REQUIRE(count >= 0 && cols >= 0, "sum_parts: negative extent");
  if (cols == 0) return kOk;
  DIONW_REQUIRE(out && (parts || count == 0), "sum_parts: null pointer");
  DIONW_REQUIRE(ceil_div(cols, 64) < INT32_MAX, "sum_parts: too many columns");
  const dim3 grid((unsigned)ceil_div(cols, 64));
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

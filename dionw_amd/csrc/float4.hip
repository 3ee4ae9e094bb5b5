// 4-bit floating-point matrices with a scale for each block of 32: quantization and reading back.
//
// A quantized matrix holds e2m1 codes (a sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6) row-major, two a
// byte, the first in its low half, its columns padded with zeros to a multiple of 256, and for every
// row and block of 32 columns the exponent byte of a float32 power of two (255: the block is NaN).
// Scaling by powers of two rounds nothing, and the matrix instructions multiply by them on the way.
// Bytes are kept by column block, [blocks][rows], so that the rows of a tile lie side by side.
//
// A weight's bytes are equal within each 32 x 32 tile, so that its transpose holds the same values;
// an activation's or a gradient's differ from row to row. Gradients are rounded stochastically: to
// nearest, what is smaller than a quarter of its block's step is lost from every sum, in 4 bits a
// large part of a gradient; up or down by chance the sums over many rows stay right on average.
#include "float4.h"

namespace dionw {
namespace {

// The most workgroups of 256 a launch takes (2^32 threads).
constexpr int64_t kMostGroups = (int64_t{1} << 24) - 1;

struct Output {
  uint8_t* data;  // null: not asked for
  int64_t ld;     // bytes
  uint8_t* scale;
  int64_t scale_ld;
};
struct QuantizeArgs {
  const void* x;
  int64_t rows, cols, ld;
  Output by_row, by_col;  // x, and its transpose
  float* sums;            // [tiles of 128 rows][cols]: each tile's column sums, or null
  int32_t tiles_c;
  int32_t far;            // 2^32 pairs of columns or more
  Noise noise;
};

// ---- by rows and by columns ----------------------------------------------------------
//
// A workgroup takes a 128 x 128 tile: thread t the rows 8 (t / 16) .. + 7 and the columns
// 8 (t % 16) .. + 7, read once and held as they are. A wave then holds 32 rows of 128 columns, so
// that every block of either form is a wave's own: 4 lanes side by side hold a row's block, 4 of a
// column of lanes a column's. Codes by rows go from registers to memory, those of the transpose
// through LDS, each in 64-byte runs; the scales through LDS, so that a block's rows are written
// together. Tiles past the last row or column, up to the padding of the other form, write zeros.
// Bound: HBM, 2 or 4 bytes read and half a byte written for each form an element; by chance, the hash and
// the conversions too. us (and TB/s) of both forms, bfloat16: 8192 x 14336 77 (4.7), by chance 88; 8192 x
// 4096 18.0 (5.7), 28; float32 8192 x 14336 133 (4.5), 14336 x 4096 by tiles 50 (5.9). Not kept: tiles
// of 256 x 128 or 256 x 256, whose runs are twice as long (79 and 81 us for the first, 34 and 42 where
// 128 x 128 took 25 by chance), and two rows of tiles in turn on one XCD (79). By chance with small
// 16-bit values cut at 2^-23 and not rounded there 80 and 25; with the definition's own arithmetic, an integer addition
// below the place kept, 116.
enum Rounding : int { kRows = 0, kTiles = 1, kStochastic = 2 };


struct Shared {
  // Words of the transpose: 17 a column, so that a wave's writes spread over the banks.
  static constexpr int pitch = 17;
  uint32_t turned[kTile4 * pitch];
  float col_sum[4][kTile4];
  __attribute__((aligned(16))) uint8_t row_bytes[4][kTile4], col_bytes[4][kTile4];
};

// Codes of a row or a column of a Square by chance, from each value's bits at the top of a word.
template <typename T, typename V, typename N>
__device__ __forceinline__ uint32_t noisy_codes(uint32_t byte, V value, N noise) {
  const float scale = power(byte), inverse = inverse4(byte);
  f32x2 p[4];
  uint32_t bits[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    p[e >> 1][e & 1] = scaled4<T>(value(e), scale, inverse);
    bits[e] = noise(e);
  }
  return noisy8(p, bits);
}

template <typename T, int ROUNDING>
__device__ __forceinline__ void quantize_tile(const QuantizeArgs& q, uint32_t tile, Shared& shared) {
  using S = Square<T>;
  constexpr int RM = S::kRowMost, CM = S::kColMost, kPitch = Shared::pitch;
  constexpr bool TILES = ROUNDING == kTiles, NOISY = ROUNDING == kStochastic;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t r0 = (int64_t)(tile / q.tiles_c) * kTile4;
  const int64_t c0 = (int64_t)(tile % q.tiles_c) * kTile4;
  const int tr = wave * 32 + lane / 16 * 8, tc = lane % 16 * 8;  // the thread's first row and column
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
  uint32_t row[RM], col[CM], tile_byte = 0;
  v.maxima(row, col);
  if (TILES) {
    uint32_t most = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) most = max(most, S::bits(col, k));
    most = largest_of_four(most);
    most = max(most, (uint32_t)__shfl_xor((int)most, 16, kWave));
    most = max(most, (uint32_t)__shfl_xor((int)most, 32, kWave));
    tile_byte = scale_byte4<false>(most);
  } else {
#pragma unroll
    for (int i = 0; i < RM; ++i) {
      row[i] = S::larger(row[i], (uint32_t)__builtin_amdgcn_update_dpp(0, (int)row[i], 0xB1, 0xF, 0xF, false));
      row[i] = S::larger(row[i], (uint32_t)__builtin_amdgcn_update_dpp(0, (int)row[i], 0x4E, 0xF, 0xF, false));
    }
    if (q.by_col.data) {
#pragma unroll
      for (int k = 0; k < CM; ++k) {
        col[k] = S::larger(col[k], (uint32_t)__shfl_xor((int)col[k], 16, kWave));
        col[k] = S::larger(col[k], (uint32_t)__shfl_xor((int)col[k], 32, kWave));
      }
    }
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
    if (lane < 16)
#pragma unroll
      for (int k = 0; k < 8; ++k) shared.col_sum[wave][tc + k] = s[k];
  }
  uint32_t h[8][4];
  if constexpr (NOISY) {
    const uint32_t key = noise_key(q.noise), near = mix32(key);
    const int64_t pairs = (q.cols + 1) / 2;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t p = (r0 + tr + i) * pairs + (c0 + tc) / 2;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        h[i][k] = mix32((uint32_t)(p + k) ^ (q.far ? mix32(key + (uint32_t)((p + k) >> 32)) : near));
    }
  }
  // Value (i, k)'s bits, at the top of a word.
  auto noise = [&](int i, int k) { return k & 1 ? h[i][k >> 1] << 16 : h[i][k >> 1]; };
  if (q.by_row.data) {
    uint8_t* out = q.by_row.data + (r0 + tr) * q.by_row.ld + (c0 + tc) / 2;
#pragma unroll
    for (int i = 0; i < 8; ++i, out += q.by_row.ld) {
      const uint32_t byte = TILES ? tile_byte : scale_byte4<NOISY>(S::bits(row, i));
      uint32_t w;
      if constexpr (NOISY) {
        w = noisy_codes<T>(byte, [&](int k) { return v.value(i, k); }, [&](int k) { return noise(i, k); });
      } else {
        w = Codes<T>::row(v, i, power(byte));
      }
      if (r0 + tr + i < q.rows) *reinterpret_cast<uint32_t*>(out) = w;
      if (lane % 4 == 0) shared.row_bytes[tc / 32][tr + i] = (uint8_t)byte;
    }
  }
  if (q.by_col.data) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t byte = TILES ? tile_byte : scale_byte4<NOISY>(S::bits(col, k));
      uint32_t w;
      if constexpr (NOISY) {
        w = noisy_codes<T>(byte, [&](int i) { return v.value(i, k); }, [&](int i) { return noise(i, k); });
      } else {
        w = Codes<T>::col(v, k, power(byte));
      }
      shared.turned[(tc + k) * kPitch + tr / 8] = w;
      if (lane < 16) shared.col_bytes[wave][tc + k] = (uint8_t)byte;
    }
  }
  __syncthreads();
  // Tiles past the last row, where the transpose is padded by more than one, have no sums.
  if (q.sums && r0 < q.rows && tid < kTile4 && c0 + tid < q.cols)
    q.sums[r0 / kTile4 * q.cols + c0 + tid] = (shared.col_sum[0][tid] + shared.col_sum[1][tid]) +
                                              (shared.col_sum[2][tid] + shared.col_sum[3][tid]);
  // A block's bytes run to a multiple of 16: 4 of them a thread, the first 128 threads the rows'.
  const int block = tid / 32 % 4, place = tid % 32 * 4;
  const Output& o = tid < 128 ? q.by_row : q.by_col;
  const int64_t first = tid < 128 ? r0 : c0, other = tid < 128 ? c0 : r0;
  if (o.data && first + place < o.scale_ld)
    *reinterpret_cast<uint32_t*>(o.scale + (other / kBlock4 + block) * o.scale_ld + first + place) =
        *reinterpret_cast<const uint32_t*>((tid < 128 ? shared.row_bytes[block] : shared.col_bytes[block]) + place);
  if (!q.by_col.data) return;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int c = j * 64 + tid / 4, word = tid % 4 * 4;
    if (c0 + c >= q.cols) continue;
    u32x4 w;
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = shared.turned[c * kPitch + word + k];
    *reinterpret_cast<u32x4*>(q.by_col.data + (c0 + c) * q.by_col.ld + r0 / 2 + 4 * word) = w;
  }
}

template <typename T, int ROUNDING>
__global__ __launch_bounds__(256) void float4_quantize_kernel(QuantizeArgs q) {
  __shared__ Shared shared;
  quantize_tile<T, ROUNDING>(q, blockIdx.x, shared);
}

// What a linear layer's forward pass quantizes, in one launch: a small layer's parts hide each
// other's latency.
template <typename TX, typename TW>
__global__ __launch_bounds__(256) void float4_quantize_pair_kernel(QuantizeArgs x, QuantizeArgs w,
                                                                   uint32_t x_tiles) {
  __shared__ Shared shared;
  if (blockIdx.x < x_tiles)
    quantize_tile<TX, kRows>(x, blockIdx.x, shared);
  else
    quantize_tile<TW, kTiles>(w, blockIdx.x - x_tiles, shared);
}

// ---- by rows alone ---------------------------------------------------------------------
//
// A workgroup takes 8 R rows of 256 columns, 32 lanes a row, 8 columns a lane: nothing goes through
// LDS but the scales. Few rows take R = 1, so that they still fill the GPU.
// Bound: HBM. bfloat16 8192 x 14336 44 us (6.7 TB/s), 8192 x 4096 13.8; float32 8192 x 14336 96 (5.5).
template <typename T, int R>
__global__ __launch_bounds__(256) void float4_quantize_rows_kernel(QuantizeArgs q) {
  __shared__ __attribute__((aligned(16))) uint8_t bytes[8][8 * R];
  const int tid = threadIdx.x, lane = tid & 31, y = tid >> 5;
  const int64_t r0 = (int64_t)(blockIdx.x / q.tiles_c) * (8 * R);
  const int64_t stage = blockIdx.x % q.tiles_c, c = stage * kDepth4 + 8 * lane;
  Square<T> v;  // R of its rows
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int64_t row = r0 + 8 * i + y;
    const T* at = reinterpret_cast<const T*>(q.x) + row * q.ld + c;
    if (row < q.rows && c + 8 <= q.cols) v.load(i, at);
    else v.load(i, at, row < q.rows ? q.cols - c : 0);
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    uint32_t most = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) most = max(most, __float_as_uint(v.value(i, k)) & 0x7FFFFFFFu);
    const uint32_t byte = scale_byte4<false>(largest_of_four(most));
    const uint32_t w = Codes<T>::row(v, i, power(byte));
    const int64_t row = r0 + 8 * i + y;
    if (row < q.rows) *reinterpret_cast<uint32_t*>(q.by_row.data + row * q.by_row.ld + c / 2) = w;
    if (lane % 4 == 0) bytes[lane / 4][8 * i + y] = (uint8_t)byte;
  }
  __syncthreads();
  if (tid < 16 * R) {  // 4 rows' bytes of a block a thread
    const int b = tid / (2 * R), place = tid % (2 * R) * 4;
    if (r0 + place < q.by_row.scale_ld)
      *reinterpret_cast<uint32_t*>(q.by_row.scale + (stage * 8 + b) * q.by_row.scale_ld + r0 + place) =
          *reinterpret_cast<const uint32_t*>(bytes[b] + place);
  }
}

// ---- reading back ------------------------------------------------------------------------
//
// The float32 values: a workgroup takes 32 rows of 256 columns, a wave 8 rows, 4 columns a lane, so
// that a wave's store is one run of 1 KB; the scales come through LDS, as a lane's rows lie together
// there.
// Bound: HBM, half a byte read and 4 written an element. 8192 x 14336 76 us (7.0 TB/s), with 8 columns a
// lane in two stores of 16 bytes 115 to 135.
struct ValuesArgs {
  const uint8_t* data;
  const uint8_t* scale;
  int64_t scale_ld, rows, cols, depth;
  float* out;
  int32_t stages;
};
__global__ __launch_bounds__(256) void float4_values_kernel(ValuesArgs g) {
  __shared__ uint8_t bytes[8][32];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t r0 = (int64_t)(blockIdx.x / g.stages) * 32, stage = blockIdx.x % g.stages;
  const int64_t c = stage * kDepth4 + 4 * lane;
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t row = min(r0 + 8 * wave + i, g.rows - 1);
    w[i] = *reinterpret_cast<const uint16_t*>(g.data + row * (g.depth / 2) + c / 2);
  }
  bytes[tid >> 5][tid & 31] =
      r0 + (tid & 31) < g.rows ? g.scale[(stage * 8 + (tid >> 5)) * g.scale_ld + r0 + (tid & 31)] : 0;
  __syncthreads();
  if (c >= g.cols) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t row = r0 + 8 * wave + i;
    if (row >= g.rows) return;
    const uint32_t byte = bytes[lane / 8][8 * wave + i];
    const float scale = byte == 255 ? __uint_as_float(0x7FC00000u) : power(byte);
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], 1.f, 0);
    const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], 1.f, 1);
    const f32x4 v = {a[0] * scale, a[1] * scale, b[0] * scale, b[1] * scale};
    float* to = g.out + row * g.cols + c;
    if (c + 4 <= g.cols) {
      typedef float f4any __attribute__((ext_vector_type(4), aligned(4)));
      __builtin_nontemporal_store(v, reinterpret_cast<f4any*>(to));
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (c + k < g.cols) to[k] = v[k];
    }
  }
}

// ---- launches ------------------------------------------------------------------------------

template <typename T>
int launch_rows(QuantizeArgs q, hipStream_t stream) {
  q.tiles_c = (int32_t)(q.by_row.ld * 2 / kDepth4);
  const int64_t most = ceil_div(q.rows, 8) * q.tiles_c;
  const bool few = most < 2048;
  const int64_t grid = ceil_div(q.rows, few ? 8 : 32) * q.tiles_c;
  DIONW_REQUIRE(grid <= kMostGroups, "float4_quantize: too many tiles");
  if (few)
    hipLaunchKernelGGL((float4_quantize_rows_kernel<T, 1>), dim3((unsigned)grid), dim3(256), 0, stream, q);
  else
    hipLaunchKernelGGL((float4_quantize_rows_kernel<T, 4>), dim3((unsigned)grid), dim3(256), 0, stream, q);
  return check_launch("float4_quantize_rows");
}

template <typename T>
int launch_quantize(const QuantizeArgs& q, int rounding, int64_t tiles, hipStream_t stream) {
  if (rounding == kRows && !q.by_col.data && !q.sums) return launch_rows<T>(q, stream);
  const dim3 grid((unsigned)tiles);
  if (rounding == kRows)
    hipLaunchKernelGGL((float4_quantize_kernel<T, kRows>), grid, dim3(256), 0, stream, q);
  else if (rounding == kTiles)
    hipLaunchKernelGGL((float4_quantize_kernel<T, kTiles>), grid, dim3(256), 0, stream, q);
  else
    hipLaunchKernelGGL((float4_quantize_kernel<T, kStochastic>), grid, dim3(256), 0, stream, q);
  return check_launch("float4_quantize");
}

bool good_elem(int32_t e) { return e == kF16 || e == kBF16 || e == kF32; }

// Checks a quantization; `tiles`: its workgroups, 0 where there is nothing to do.
int prepare(const Quantization4& j, QuantizeArgs& q, int64_t& tiles) {
  tiles = 0;
  DIONW_REQUIRE(good_elem(j.elem), "float4_quantize: bad element type %d", j.elem);
  DIONW_REQUIRE(j.rows >= 0 && j.cols >= 0, "float4_quantize: negative extent");
  if (j.rows == 0 || j.cols == 0) return kOk;
  DIONW_REQUIRE(j.by_row.data || j.by_col.data || j.sums, "float4_quantize: no output");
  DIONW_REQUIRE(j.x && j.ld >= j.cols, "float4_quantize: bad input");
  auto fits = [](const Matrix4& o, int64_t r, int64_t c) {
    return !o.data || (o.depth == round_up(c, kDepth4) && aligned16(o.data) && o.scale && o.scale_ld >= r &&
                       o.scale_ld % 16 == 0 && aligned16(o.scale));
  };
  DIONW_REQUIRE(fits(j.by_row, j.rows, j.cols) && fits(j.by_col, j.cols, j.rows),
                "float4_quantize: an output is too small or not aligned");
  const int64_t tr = ceil_div(j.by_col.data ? j.by_col.depth : j.rows, kTile4);
  const int64_t tc = ceil_div(j.by_row.data ? j.by_row.depth : j.cols, kTile4);
  DIONW_REQUIRE(tr <= kMostGroups / tc, "float4_quantize: too many tiles");
  auto output = [](const Matrix4& o) {
    return Output{static_cast<uint8_t*>(o.data), o.depth / 2, static_cast<uint8_t*>(o.scale), o.scale_ld};
  };
  q = {};
  q.x = j.x;
  q.rows = j.rows;
  q.cols = j.cols;
  q.ld = j.ld;
  q.by_row = output(j.by_row);
  q.by_col = output(j.by_col);
  q.sums = j.sums;
  q.tiles_c = (int32_t)tc;
  q.far = tr * kTile4 > (int64_t{1} << 32) / (tc * kTile4 / 2);
  tiles = tr * tc;
  return kOk;
}

template <typename TX>
int launch_pair(const QuantizeArgs& x, int64_t x_tiles, int32_t w_elem, const QuantizeArgs& w,
                int64_t w_tiles, hipStream_t stream) {
  const dim3 grid((unsigned)(x_tiles + w_tiles));
  auto launch = [&](auto kern) {
    hipLaunchKernelGGL(kern, grid, dim3(256), 0, stream, x, w, (uint32_t)x_tiles);
  };
  if (w_elem == kF16) launch(float4_quantize_pair_kernel<TX, _Float16>);
  else if (w_elem == kBF16) launch(float4_quantize_pair_kernel<TX, __bf16>);
  else launch(float4_quantize_pair_kernel<TX, float>);
  return check_launch("float4_quantize_pair");
}

}  // namespace

int quantize4(const Quantization4& x, bool tiles, const Noise* noise, hipStream_t stream) {
  QuantizeArgs q{};
  int64_t count;
  DIONW_REQUIRE(!(tiles && noise), "float4_quantize: tiles are rounded to nearest");
  DIONW_TRY(prepare(x, q, count));
  if (count == 0) return kOk;
  if (noise) q.noise = *noise;
  const int rounding = noise ? kStochastic : tiles ? kTiles : kRows;
  if (x.elem == kF16) return launch_quantize<_Float16>(q, rounding, count, stream);
  if (x.elem == kBF16) return launch_quantize<__bf16>(q, rounding, count, stream);
  return launch_quantize<float>(q, rounding, count, stream);
}

int quantize4_pair(const Quantization4& x, const Quantization4& w, hipStream_t stream) {
  QuantizeArgs qx{}, qw{};
  int64_t x_tiles, w_tiles;
  DIONW_TRY(prepare(x, qx, x_tiles));
  DIONW_TRY(prepare(w, qw, w_tiles));
  if (x_tiles + w_tiles == 0) return kOk;
  DIONW_REQUIRE(x_tiles + w_tiles <= kMostGroups, "float4_quantize: too many tiles");
  if (x.elem == kF16) return launch_pair<_Float16>(qx, x_tiles, w.elem, qw, w_tiles, stream);
  if (x.elem == kBF16) return launch_pair<__bf16>(qx, x_tiles, w.elem, qw, w_tiles, stream);
  return launch_pair<float>(qx, x_tiles, w.elem, qw, w_tiles, stream);
}

}  // namespace dionw

using namespace dionw;

extern "C" {

int dionw_float4_quantize(int32_t elem, const void* x, int64_t rows, int64_t cols, int64_t ld,
                          int32_t rounding, int64_t seed, const int64_t* seed_at, void* data,
                          void* scale, int64_t scale_ld, void* data_t, void* scale_t,
                          int64_t scale_t_ld, hipStream_t stream) {
  DIONW_REQUIRE(rounding >= kRows && rounding <= kStochastic, "float4_quantize: bad rounding %d", rounding);
  const Noise noise{seed, seed_at};
  return quantize4({elem, x, rows, cols, ld,
                    {data, scale, rows, round_up(cols, kDepth4), scale_ld},
                    {data_t, scale_t, cols, round_up(rows, kDepth4), scale_t_ld}, nullptr},
                   rounding == kTiles, rounding == kStochastic ? &noise : nullptr, stream);
}

int dionw_float4_values(const void* data, const void* scale, int64_t scale_ld, int64_t rows,
                        int64_t cols, float* out, hipStream_t stream) {
  DIONW_REQUIRE(rows >= 0 && cols >= 0, "float4_values: negative extent");
  if (rows == 0 || cols == 0) return kOk;
  DIONW_REQUIRE(data && scale && out && aligned16(data) && scale_ld >= rows,
                "float4_values: a matrix is too small or not aligned");
  const int64_t depth = round_up(cols, kDepth4), stages = depth / kDepth4;
  DIONW_REQUIRE(ceil_div(rows, 32) <= kMostGroups / stages, "float4_values: too many elements");
  const ValuesArgs g{static_cast<const uint8_t*>(data), static_cast<const uint8_t*>(scale), scale_ld, rows,
                     cols, depth, out, (int32_t)stages};
  hipLaunchKernelGGL(float4_values_kernel, dim3((unsigned)(ceil_div(rows, 32) * stages)), dim3(256), 0, stream, g);
  return check_launch("float4_values");
}

}  // extern "C"

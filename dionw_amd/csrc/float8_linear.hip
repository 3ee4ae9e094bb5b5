// The linear layer on 8-bit operands: its passes in order, with their scratch laid out here, and
// the product of a few rows with a kept weight.
#include "float8.h"

#include <type_traits>

namespace dionw {
namespace {

// ---- a few rows ----------------------------------------------------------------------
//
// y = x W^T + b for 16 rows of x at a time (the tokens being decoded): every byte of W passes
// once, from memory to registers, and x is quantized on the way, so that the call is one launch.
// A workgroup takes 16 R rows of W; its waves take the blocks of 128 columns in turn and add their
// sums through LDS, in a fixed order. Of a block, a lane holds one token's (or weight row's)
// chunks of 16 at places G = lane / 16 and 4 + G, so that each load of a wave covers 64 bytes of
// 16 rows; the block's largest magnitude is one of 4 lanes', two exchanges. A wave reads the next
// block while it multiplies one.
// Bound: HBM, n k bytes of W; the smallest calls: launch and the latency of two dependent reads.
//
// 16-bit calls of more rows quantize x first and go through the tiles. float32 ones would expand W
// for that, 5 bytes of traffic for each of its codes, so they run as groups of 16 here up to 32
// rows, and up to 64 of at most 4096 columns, each group reading W again. us for 64 rows here / 65
// through the tiles: 4096 x 1024 7.5 / 16, 4096 x 4096 19 / 27, 14336 x 4096 70 / 61, 28672 x 4096 126 /
// 136; 1024 x 14336 34 / 28, 4096 x 14336 60 / 61, 6144 x 14336 122 / 87, 14336 x 14336 248 / 228. For 32
// rows here, of 14336 columns: 34, 46, 61, 125.
constexpr int kFew = 16, kFewFloat = 32, kFewFloatShallow = 64, kShallow = 4096;
bool few_rows(int32_t elem, int64_t m, int64_t k) {
  return k > 0 && m <= (elem != kF32 ? kFew : k <= kShallow ? kFewFloatShallow : kFewFloat);
}

struct FewArgs {
  const void* x;
  int64_t x_ld;
  const uint8_t* w;
  int64_t w_ld;
  const uint8_t* w_scale;
  int64_t w_scale_ld;
  const float* bias;
  void* y;
  int64_t k;
  int32_t m, n, blocks;
};

// 32 values of a token's block, as they lie in memory.
template <typename T>
struct Values {
  static constexpr int kWords = 8 * sizeof(T);
  uint32_t w[kWords];
  // `left`: columns from the block's first one on, at least 1 (WHOLE: 128).
  template <bool WHOLE>
  __device__ __forceinline__ void load(const T* block, int G, int left) {
    constexpr int kHalf = kWords / 2;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = 64 * h + 16 * G;
      if constexpr (WHOLE) {
#pragma unroll
        for (int v = 0; v < kHalf / 4; ++v) {
          const u32x4 r = *reinterpret_cast<const u32x4_any*>(block + c + 16 / sizeof(T) * v);
#pragma unroll
          for (int e = 0; e < 4; ++e) w[h * kHalf + 4 * v + e] = r[e];
        }
      } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const uint32_t v = __float_as_uint(block[min(c + e, left - 1)]);
          w[h * kHalf + e] = c + e < left ? v : 0u;
        }
      } else {
        const uint16_t* u = reinterpret_cast<const uint16_t*>(block);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t lo = u[min(c + 2 * e, left - 1)], hi = u[min(c + 2 * e + 1, left - 1)];
          w[h * kHalf + e] = (c + 2 * e < left ? lo : 0u) | (c + 2 * e + 1 < left ? hi : 0u) << 16;
        }
      }
    }
  }
  // The float32 bits of the largest finite magnitude.
  __device__ __forceinline__ uint32_t most() const {
    uint32_t m = 0;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < kWords; ++i) m = max(m, w[i] & 0x7FFFFFFFu);
      if (m >= 0x7F800000u) {
        m = 0;
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
          const uint32_t b = w[i] & 0x7FFFFFFFu;
          m = max(m, b < 0x7F800000u ? b : 0u);
        }
      }
      return m;
    } else {
      using P = Pair<T>;
#pragma unroll
      for (int i = 0; i < kWords; ++i) m = P::larger(m, w[i] & 0x7FFF7FFFu);
      m = max(m & 0xFFFFu, m >> 16);
      if (m >= P::inf) {
        m = 0;
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
          const uint32_t lo = w[i] & 0x7FFFu, hi = w[i] >> 16 & 0x7FFFu;
          m = max(m, max(lo < P::inf ? lo : 0u, hi < P::inf ? hi : 0u));
        }
      }
      return P::bits(m);
    }
  }
  __device__ __forceinline__ i32x8 codes(float scale) const {
    i32x8 c;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (sizeof(T) == 4)
        c[i] = (int)codes4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3], scale);
      else
        c[i] = (int)codes4(w[2 * i], w[2 * i + 1], scale, T{});
    }
    return c;
  }
};

template <typename T, int R, int W, bool WHOLE>
__global__ __launch_bounds__(W * 64) void float8_few_kernel(FewArgs g) {
  constexpr bool kExact = std::is_same<T, float>::value;  // float32 sums on expanded codes
  __shared__ f32x4 sums[W][R][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int G = lane >> 4, i16 = lane & 15;
  const int n0 = blockIdx.x * 16 * R, token = blockIdx.y * 16 + i16;
  const T* x = reinterpret_cast<const T*>(g.x) + min(token, g.m - 1) * g.x_ld;
  const uint8_t* w[R];
  int row[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    row[r] = min(n0 + 16 * r + i16, g.n - 1);
    w[r] = g.w + row[r] * g.w_ld + 16 * G;
  }
  struct Block {
    Values<T> x;
    i32x4 w[R][2];
    uint32_t byte[R];
  };
  auto read = [&](Block& b, int kb) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      b.w[r][0] = __builtin_nontemporal_load(reinterpret_cast<const i32x4*>(w[r] + (int64_t)kb * kTile));
      b.w[r][1] = __builtin_nontemporal_load(reinterpret_cast<const i32x4*>(w[r] + (int64_t)kb * kTile + 64));
      b.byte[r] = g.w_scale[kb * g.w_scale_ld + row[r]];
    }
    if (WHOLE || kb < g.blocks - 1)
      b.x.template load<true>(x + (int64_t)kb * kTile, G, kTile);
    else
      b.x.template load<false>(x + (int64_t)kb * kTile, G, (int)(g.k - (int64_t)kb * kTile));
  };
  f32x4 acc[R];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[r][e] = 0.f;
  auto multiply = [&](Block& b) {
    uint32_t most = b.x.most();
    most = max(most, (uint32_t)__shfl_xor((int)most, 16, kWave));
    most = max(most, (uint32_t)__shfl_xor((int)most, 32, kWave));
    const uint32_t byte = scale_byte(most);
    const i32x8 c = b.x.codes(power(byte));
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const i32x8 v = __builtin_shufflevector(b.w[r][0], b.w[r][1], 0, 1, 2, 3, 4, 5, 6, 7);
      if constexpr (kExact) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          acc[r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              expand(v[2 * q], v[2 * q + 1], half_power(b.byte[r])),
              expand(c[2 * q], c[2 * q + 1], half_power(byte)), acc[r], 0, 0, 0);
      } else {
        acc[r] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(v, c, acc[r], 0, 0, 0, b.byte[r], 0, byte);
      }
    }
  };
  Block a, b;
  int kb = wave;
  if (kb < g.blocks) read(a, kb);
  for (; kb < g.blocks; kb += 2 * W) {
    if (kb + W < g.blocks) read(b, kb + W);
    multiply(a);
    if (kb + W >= g.blocks) break;
    if (kb + 2 * W < g.blocks) read(a, kb + 2 * W);
    multiply(b);
  }
#pragma unroll
  for (int r = 0; r < R; ++r) sums[wave][r][lane] = acc[r];
  __syncthreads();
  for (int t = wave; t < R; t += W) {  // a fragment a wave: lane: token i16, rows 4 G .. + 3 of W
    f32x4 s = sums[0][t][lane];
#pragma unroll
    for (int v = 1; v < W; ++v) s += sums[v][t][lane];
    const int n = n0 + 16 * t + 4 * G;
    if (token >= g.m || n >= g.n) continue;
    typedef T t4 __attribute__((ext_vector_type(4)));
    typedef T t4any __attribute__((ext_vector_type(4), aligned(sizeof(T))));
    t4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      o[e] = (T)((kExact ? kExpanded : 1.f) * s[e] + (g.bias ? g.bias[min(n + e, g.n - 1)] : 0.f));
    T* y = reinterpret_cast<T*>(g.y) + (int64_t)token * g.n + n;
    if (n + 4 <= g.n) {
      *reinterpret_cast<t4any*>(y) = o;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < g.n) y[e] = o[e];
    }
  }
}

// R rows' fragments a wave and W waves a workgroup: many fragments (counted for each group of 16
// tokens) take 64 rows each (x is read and quantized once for them), few the most workgroups. us in
// a chain of launches (an empty one takes 4), R W = 1 8 / 2 8 / 4 4, bfloat16, a row of x: 1024 x 4096
// 5.3 / 8.1 / 13.5, 4096 x 4096 6.8 / 8.7 / 14.1, 4096 x 14336 15.0 / 24.3 / 41.5, 6144 x 4096 9.6 / 9.2 / 14.4,
// 8192 x 4096 10.5 / 9.9 / 14.8, 10240 x 4096 13.3 / 14.9 / 15.2, 14336 x 4096 (8 rows of x) 20.4 / 17.4 /
// 16.7, 128256 x 4096 112 / 100 / 96, with 16 rows 181 / 138 / 119. The type counts between 512 and 768
// fragments alone, 10240 x 4096: 16 bits, 16 rows 20.1 / 19.3 / 16.6, 8 16.5 / 16.9 / 15.7 (the number
// of rows is not asked, so that a row's sums do not depend on the rows beside it); float32, 1 row
// 19.6 / 18.7 / 16.3, 16 33 / 29 / 20. float32 groups: 2 of 4096 x 4096 23 / 15.5 / 19, 2 of 8192 x 4096 44 /
// 30 / 20, 4 of 4096 x 14336 135 / 91 / 60, 4 of 28672 x 4096 294 / 195 / 126.
template <typename T, bool WHOLE>
int launch_few(const FewArgs& g, hipStream_t stream) {
  const int fragments = (g.n + 15) / 16;
  const unsigned groups = (unsigned)(g.m + 15) / 16;
  const int64_t all = (int64_t)fragments * groups;
  if (all < 320 || (sizeof(T) == 2 && all > 512 && all < 768))
    hipLaunchKernelGGL((float8_few_kernel<T, 1, 8, WHOLE>), dim3(fragments, groups), dim3(512), 0, stream, g);
  else if (all <= 512)
    hipLaunchKernelGGL((float8_few_kernel<T, 2, 8, WHOLE>), dim3((fragments + 1) / 2, groups), dim3(512), 0, stream, g);
  else
    hipLaunchKernelGGL((float8_few_kernel<T, 4, 4, WHOLE>), dim3((fragments + 3) / 4, groups), dim3(256), 0, stream, g);
  return check_launch("float8_few");
}

// WHOLE: the depth is a multiple of 128, so that no block needs its columns counted.
template <typename T>
int launch_few(const FewArgs& g, hipStream_t stream) {
  return g.k % kTile ? launch_few<T, false>(g, stream) : launch_few<T, true>(g, stream);
}

// ---- scratch ---------------------------------------------------------------------------

// Hands out parts of a buffer (of nothing, where only sizes are asked for).
struct Parts {
  uint8_t* base;
  size_t used = 0;
  void* take(size_t bytes) {
    void* at = base ? base + used : nullptr;
    used += round_up((int64_t)bytes, 256);
    return at;
  }
};

Matrix codes_in(Parts& p, int64_t rows, int64_t cols) {
  Matrix q{nullptr, nullptr, rows, round_up(cols, kTile), round_up(rows, 16)};
  q.data = p.take((size_t)(rows * q.depth));
  q.scale = p.take((size_t)(q.depth / kTile * q.scale_ld));
  return q;
}
Matrix expanded_in(Parts& p, int64_t rows, int64_t cols) {
  Matrix q{nullptr, nullptr, rows, round_up(cols, kTile), 0};
  q.data = p.take((size_t)(rows * q.depth) * 2);
  return q;
}
Matrix operand_in(Parts& p, bool expanded, int64_t rows, int64_t cols) {
  return expanded ? expanded_in(p, rows, cols) : codes_in(p, rows, cols);
}

struct Saved {
  Matrix wt, xt;
  Saved(Parts& p, int64_t m, int64_t n, int64_t k, bool need_x, bool need_w) : wt{}, xt{} {
    if (need_x) wt = codes_in(p, k, n);
    if (need_w) xt = codes_in(p, k, m);
  }
};

struct Forward {
  Matrix x, w;
  void* product;
  size_t product_bytes;
  Forward(Parts& p, bool exact, int64_t m, int64_t n, int64_t k) {
    x = operand_in(p, exact, m, k);
    w = operand_in(p, exact, n, k);
    product_bytes = dionw_float8_gemm_workspace(exact, m, n, x.depth);
    product = p.take(product_bytes);
  }
};

struct Backward {
  Matrix rows{}, cols{}, wt{}, xt{};  // dy by rows and columns; W's and x's transposes, expanded
  float* sums = nullptr;
  size_t product_bytes = 0;
  void* product;
  Backward(Parts& p, bool exact_x, bool exact_w, int64_t m, int64_t n, int64_t k, bool need_x,
           bool need_w, bool need_b) {
    if (need_x) {
      rows = operand_in(p, exact_x, m, n);
      if (exact_x) wt = expanded_in(p, k, n);
      product_bytes = dionw_float8_gemm_workspace(exact_x, m, k, rows.depth);
    }
    if (need_w) {
      cols = operand_in(p, exact_w, n, m);
      if (exact_w) xt = expanded_in(p, k, m);
      const size_t bytes = dionw_float8_gemm_workspace(exact_w, n, k, cols.depth);
      if (bytes > product_bytes) product_bytes = bytes;
    }
    if (need_b) sums = static_cast<float*>(p.take((size_t)(ceil_div(m, kTile) * n) * 4));
    product = p.take(product_bytes);
  }
};

int product(bool expanded, const Matrix& a, const Matrix& b, const float* bias, int32_t elem, void* c,
            void* space, size_t bytes, hipStream_t stream) {
  return dionw_float8_gemm(expanded, a.rows, b.rows, a.depth, a.data, a.depth, a.scale, a.scale_ld,
                           b.data, b.depth, b.scale, b.scale_ld, bias, elem, c, b.rows, space, bytes,
                           stream);
}

// Whether an operand of that many columns is one the products take, for results of type `elem`.
bool fits_row(int64_t cols, int32_t elem) {
  return cols < kRowBytes && round_up(cols, kTile) * (elem == kF32 ? 2 : 1) < kRowBytes;
}

bool good_elem(int32_t e) { return e == kF16 || e == kBF16 || e == kF32; }

}  // namespace
}  // namespace dionw

using namespace dionw;

extern "C" {

void dionw_float8_linear_sizes(int32_t x_elem, int32_t w_elem, int64_t m, int64_t n, int64_t k,
                               int32_t need_x, int32_t need_w, int32_t need_b, size_t* sizes) {
  Parts saved{nullptr}, forward{nullptr}, backward{nullptr};
  Saved s(saved, m, n, k, need_x, need_w);
  Forward f(forward, x_elem == kF32, m, n, k);
  Backward b(backward, x_elem == kF32, w_elem == kF32, m, n, k, need_x, need_w, need_b);
  sizes[0] = saved.used;
  sizes[1] = forward.used;
  sizes[2] = backward.used;
}

int dionw_float8_linear_forward(int32_t x_elem, const void* x, int64_t x_ld, int32_t w_elem,
                                const void* w, int64_t w_ld, const float* bias, int64_t m,
                                int64_t n, int64_t k, int32_t need_x, int32_t need_w, void* y,
                                void* saved, void* scratch, size_t scratch_bytes,
                                hipStream_t stream) {
  DIONW_REQUIRE(good_elem(x_elem) && good_elem(w_elem), "float8_linear: bad element type");
  DIONW_REQUIRE(m >= 0 && n >= 0 && k >= 0, "float8_linear: negative extent");
  DIONW_REQUIRE(saved || !(need_x || need_w) || m == 0 || n == 0 || k == 0, "float8_linear: no room to save");
  // The gradients sum over n and m: refused here rather than after the forward pass.
  DIONW_REQUIRE((!need_x || fits_row(n, x_elem)) && (!need_w || fits_row(m, w_elem)),
                "float8_linear: a gradient's product takes rows of less than 8 MB");
  DIONW_REQUIRE(aligned16(saved) && aligned16(scratch), "float8_linear: buffers need 16-byte alignment");
  Parts kept{static_cast<uint8_t*>(saved)}, room{static_cast<uint8_t*>(scratch)};
  const bool exact = x_elem == kF32;
  Saved s(kept, m, n, k, need_x, need_w);
  Forward f(room, exact, m, n, k);
  DIONW_REQUIRE(room.used <= scratch_bytes && (scratch || room.used == 0), "float8_linear: scratch too small");
  if (m == 0) return kOk;  // y and dx are empty, dW and db sums of nothing: nothing that is saved is read
  DIONW_TRY(quantize_pair({x_elem, x, m, k, x_ld, f.x, s.xt, nullptr},
                          {w_elem, w, n, k, w_ld, f.w, s.wt, nullptr}, stream));
  return product(exact, f.x, f.w, bias, x_elem, y, f.product, f.product_bytes, stream);
}

int dionw_float8_linear_backward(int32_t x_elem, const void* dy, int64_t dy_ld, int32_t w_elem,
                                 int64_t m, int64_t n, int64_t k, int32_t need_x, int32_t need_w,
                                 const void* saved, void* dx, void* dw, int32_t bias_elem,
                                 void* db, void* scratch, size_t scratch_bytes,
                                 hipStream_t stream) {
  DIONW_REQUIRE(good_elem(x_elem) && good_elem(w_elem), "float8_linear: bad element type");
  DIONW_REQUIRE(m >= 0 && n >= 0 && k >= 0, "float8_linear: negative extent");
  DIONW_REQUIRE(aligned16(saved) && aligned16(scratch), "float8_linear: buffers need 16-byte alignment");
  Parts kept{static_cast<uint8_t*>(const_cast<void*>(saved))}, room{static_cast<uint8_t*>(scratch)};
  const bool exact_x = x_elem == kF32, exact_w = w_elem == kF32;
  Saved s(kept, m, n, k, need_x, need_w);
  Backward b(room, exact_x, exact_w, m, n, k, need_x, need_w, db != nullptr);
  DIONW_REQUIRE(room.used <= scratch_bytes && (scratch || room.used == 0), "float8_linear: scratch too small");
  DIONW_REQUIRE(saved || kept.used == 0, "float8_linear: nothing was saved");
  if (m > 0) {
    DIONW_TRY(quantize_and_expand({x_elem, dy, m, n, dy_ld, b.rows, b.cols, b.sums}, {s.wt, s.xt},
                                  {b.wt, b.xt}, stream));
  }
  if (need_x) {
    DIONW_TRY(product(exact_x, b.rows, exact_x ? b.wt : s.wt, nullptr, x_elem, dx, b.product,
                      b.product_bytes, stream));
  }
  if (need_w) {
    DIONW_TRY(product(exact_w, b.cols, exact_w ? b.xt : s.xt, nullptr, w_elem, dw, b.product,
                      b.product_bytes, stream));
  }
  return db ? dionw_sum_parts(b.sums, ceil_div(m, kTile), n, bias_elem, db, stream) : kOk;
}

size_t dionw_float8_linear_kept_scratch(int32_t x_elem, int64_t m, int64_t n, int64_t k) {
  if (few_rows(x_elem, m, k)) return 0;
  Parts room{nullptr};
  if (x_elem == kF32) {
    Forward f(room, true, m, n, k);
  } else {
    const Matrix x = codes_in(room, m, k);
    room.take(dionw_float8_gemm_workspace(0, m, n, x.depth));
  }
  return room.used;
}

int dionw_float8_linear_kept(int32_t x_elem, const void* x, int64_t x_ld, const void* w,
                             int64_t w_ld, const void* w_scale, int64_t w_scale_ld,
                             const float* bias, int64_t m, int64_t n, int64_t k, void* y,
                             void* scratch, size_t scratch_bytes, hipStream_t stream) {
  DIONW_REQUIRE(good_elem(x_elem), "float8_linear: bad element type %d", x_elem);
  DIONW_REQUIRE(m >= 0 && n >= 0 && k >= 0 && n < INT32_MAX / 2, "float8_linear: bad extents");
  if (m == 0 || n == 0) return kOk;
  const int64_t depth = round_up(k, kTile);
  DIONW_REQUIRE(y && (k == 0 || (x && w && w_scale)), "float8_linear: null pointer");
  DIONW_REQUIRE(x_ld >= k && w_ld >= depth && w_ld % 16 == 0 && aligned16(w) && w_scale_ld >= n &&
                    aligned16(scratch),
                "float8_linear: an operand is too small or not aligned");
  const Matrix weight{const_cast<void*>(w), const_cast<void*>(w_scale), n, depth, w_scale_ld};
  if (few_rows(x_elem, m, k)) {
    DIONW_REQUIRE(depth / kTile < INT32_MAX / 2, "float8_linear: depth too large");
    const FewArgs g{x, x_ld, static_cast<const uint8_t*>(w), w_ld, static_cast<const uint8_t*>(w_scale),
                    w_scale_ld, bias, y, k, (int32_t)m, (int32_t)n, (int32_t)(depth / kTile)};
    if (x_elem == kF16) return launch_few<_Float16>(g, stream);
    if (x_elem == kBF16) return launch_few<__bf16>(g, stream);
    return launch_few<float>(g, stream);
  }
  DIONW_REQUIRE(w_ld == depth, "float8_linear: a kept weight's rows lie at its depth");
  Parts room{static_cast<uint8_t*>(scratch)};
  const bool exact = x_elem == kF32;
  if (exact) {
    Forward f(room, true, m, n, k);
    DIONW_REQUIRE(room.used <= scratch_bytes, "float8_linear: scratch too small");
    DIONW_TRY(quantize_and_expand({x_elem, x, m, k, x_ld, f.x, {}, nullptr}, {weight, {}}, {f.w, {}}, stream));
    return product(true, f.x, f.w, bias, x_elem, y, f.product, f.product_bytes, stream);
  }
  const Matrix rows = codes_in(room, m, k);
  const size_t bytes = dionw_float8_gemm_workspace(0, m, n, depth);
  void* space = room.take(bytes);
  DIONW_REQUIRE(room.used <= scratch_bytes, "float8_linear: scratch too small");
  DIONW_TRY(dionw_float8_quantize(x_elem, x, m, k, x_ld, 0, rows.data, rows.depth, rows.scale, rows.scale_ld,
                                  nullptr, 0, nullptr, 0, 0, nullptr, stream));
  return product(false, rows, weight, bias, x_elem, y, space, bytes, stream);
}

}  // extern "C"

// The linear layer on 4-bit operands: its passes in order, with their scratch laid out here, and
// the product of a few rows with a kept weight.
#include "float4.h"

#include <type_traits>

namespace dionw {
namespace {

// ---- a few rows ----------------------------------------------------------------------
//
// y = x W^T + b for 16 rows of x at a time (the tokens being decoded): every byte of W passes
// once, from memory to registers, and x is quantized on the way, so that the call is one launch.
// A workgroup takes 16 R rows of W; its waves take the stages of 256 columns in turn and add their
// sums through LDS, in a fixed order. Of a stage, a lane holds one token's (or weight row's) two
// blocks of 32, number G = lane / 16 and 4 + G: a block's scale and codes are its lane's own, without
// an exchange. A wave reads the next stage while it multiplies one.
// Bound: HBM, n k (1 / 2 + 1 / 32) bytes of W: 128256 x 4096 51.4 us, 5.4 TB/s (reading the codes alone, in
// this order, 45, from end to end 39); the smallest calls: launch and the latency of two dependent reads.
constexpr int kFew = 16;
bool few_rows(int64_t m, int64_t k) { return k > 0 && m <= kFew; }

struct FewArgs {
  const void* x;
  int64_t x_ld;
  const uint8_t* w;
  const uint8_t* w_scale;
  int64_t w_scale_ld;
  const float* bias;
  void* y;
  int64_t k;
  int32_t m, n, stages;
};

// A token's block of 32 as it lies in memory, and its codes.
template <typename T>
struct Values {
  static constexpr int kWords = 8 * sizeof(T);
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const T* at) {
#pragma unroll
    for (int v = 0; v < kWords / 4; ++v) {
      const u32x4 r = *reinterpret_cast<const u32x4_any*>(at + 16 / sizeof(T) * v);
#pragma unroll
      for (int e = 0; e < 4; ++e) w[4 * v + e] = r[e];
    }
  }
  // Zeros from the `left`th value on.
  __device__ __forceinline__ void load(const T* at, int64_t left) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int e = 0; e < 32; ++e) w[e] = e < left ? __float_as_uint(at[e]) : 0u;
    } else {
      const uint16_t* u = reinterpret_cast<const uint16_t*>(at);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const uint32_t lo = 2 * e < left ? u[2 * e] : 0, hi = 2 * e + 1 < left ? u[2 * e + 1] : 0;
        w[e] = lo | hi << 16;
      }
    }
  }
  // The float32 bits of the largest magnitude.
  __device__ __forceinline__ uint32_t most() const {
    uint32_t m = 0;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < kWords; ++i) m = max(m, w[i] & 0x7FFFFFFFu);
      return m;
    } else {
      using P = Pair<T>;
#pragma unroll
      for (int i = 0; i < kWords; ++i) m = P::larger(m, w[i] & 0x7FFF7FFFu);
      return P::bits(max(m & 0xFFFFu, m >> 16));
    }
  }
  template <int B>
  __device__ __forceinline__ uint32_t pair(uint32_t old, int i, float scale) const {
    if constexpr (sizeof(T) == 4)
      return codes2<B>(old, __uint_as_float(w[8 * i + 2 * B]), __uint_as_float(w[8 * i + 2 * B + 1]), scale);
    else
      return codes2<B>(old, w[4 * i + B], scale, T{});
  }
  __device__ __forceinline__ i32x4 codes(float scale) const {
    i32x4 c;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      c[i] = (int)pair<3>(pair<2>(pair<1>(pair<0>(0, i, scale), i, scale), i, scale), i, scale);
    return c;
  }
};

// c += b a^T; b's scale is byte B of its word.
template <int B>
__device__ __forceinline__ void multiply4(i32x4 b, i32x4 a, f32x4& c, uint32_t b_scale, uint32_t a_scale) {
  c = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
      __builtin_shufflevector(b, b, 0, 1, 2, 3, -1, -1, -1, -1),
      __builtin_shufflevector(a, a, 0, 1, 2, 3, -1, -1, -1, -1), c, 4, 4, B, (int)b_scale, 0, (int)a_scale);
}

// A workgroup takes P parts of 16 R rows of W, for which x is read and quantized once.
template <typename T, int R, int P, int W, bool WHOLE>
__global__ __launch_bounds__(W * 64) void float4_few_kernel(FewArgs g) {
  __shared__ f32x4 sums[W][P][R][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int G = lane >> 4, i16 = lane & 15;
  const int n0 = blockIdx.x * 16 * R * P, token = blockIdx.y * 16 + i16;
  const T* x = reinterpret_cast<const T*>(g.x) + min(token, g.m - 1) * g.x_ld + kBlock4 * G;
  const uint8_t *w[P][R], *scale[P];
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const int n = n0 + 16 * R * p + R * i16;  // the lane's first row
#pragma unroll
    for (int r = 0; r < R; ++r) w[p][r] = g.w + (int64_t)min(n + r, g.n - 1) * g.stages * 128 + 16 * G;
    // A block's bytes run to a multiple of 16; words past the last belong to rows past it too.
    scale[p] = g.w_scale + G * g.w_scale_ld + min((int64_t)n, g.w_scale_ld - R);
  }
  using Word = std::conditional_t<R == 4, uint32_t, std::conditional_t<R == 2, uint16_t, uint8_t>>;
  struct Rows {  // a stage of a part's rows
    i32x4 w[R][2];
    uint32_t bytes[2];
  };
  auto read = [&](Rows& s, int kt, int p) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int r = 0; r < R; ++r)
        s.w[r][h] = __builtin_nontemporal_load(reinterpret_cast<const i32x4*>(w[p][r] + (int64_t)kt * 128 + 64 * h));
      s.bytes[h] = *reinterpret_cast<const Word*>(scale[p] + ((int64_t)kt * 8 + 4 * h) * g.w_scale_ld);
    }
  };
  Values<T> v[2];  // x as it comes, and its codes and scales
  i32x4 c[2];
  uint32_t byte[2];
  auto read_x = [&](int kt) {
    const int64_t at = (int64_t)kt * kDepth4;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int64_t left = g.k - at - 128 * h - kBlock4 * G;  // columns from the block's first one on
      if (WHOLE || left >= kBlock4) v[h].load(x + at + 128 * h);
      else v[h].load(x + at + 128 * h, left);
    }
  };
  f32x4 acc[P][R];
#pragma unroll
  for (int p = 0; p < P; ++p)
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[p][r][e] = 0.f;
  // Part p of stage kt, which `now` holds; what follows it is read into `next`. x goes out before the
  // rows that are multiplied by it, so that it can be quantized while they are on their way.
  auto part = [&](auto p_, int kt, const Rows& now, Rows& next) {
    constexpr int p = decltype(p_)::value;
    if constexpr (p + 1 < P) read(next, kt, p + 1);
    if constexpr (p == 0) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        byte[h] = scale_byte4<false>(v[h].most());
        c[h] = v[h].codes(power(byte[h]));
      }
      if (kt + W < g.stages) read_x(kt + W);
    }
    if constexpr (p + 1 == P)
      if (kt + W < g.stages) read(next, kt + W, 0);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      multiply4<0>(now.w[0][h], c[h], acc[p][0], now.bytes[h], byte[h]);
      if constexpr (R > 1) multiply4<1>(now.w[1][h], c[h], acc[p][1], now.bytes[h], byte[h]);
      if constexpr (R > 2) {
        multiply4<2>(now.w[2][h], c[h], acc[p][2], now.bytes[h], byte[h]);
        multiply4<3>(now.w[3][h], c[h], acc[p][3], now.bytes[h], byte[h]);
      }
    }
  };
  using I0 = std::integral_constant<int, 0>;
  using I1 = std::integral_constant<int, 1>;
  using I2 = std::integral_constant<int, 2>;
  using I3 = std::integral_constant<int, 3>;
  static_assert(P == 1 || P == 2 || P == 4, "a stage's parts begin in the same registers");
  Rows a, b;
  int kt = wave;
  if (kt < g.stages) {
    read_x(kt);
    read(a, kt, 0);
  }
  for (; kt < g.stages; kt += W) {
    part(I0{}, kt, a, b);
    if constexpr (P == 1) {
      kt += W;
      if (kt < g.stages) part(I0{}, kt, b, a);
    }
    if constexpr (P > 1) part(I1{}, kt, b, a);
    if constexpr (P > 2) {
      part(I2{}, kt, a, b);
      part(I3{}, kt, b, a);
    }
  }
#pragma unroll
  for (int p = 0; p < P; ++p)
#pragma unroll
    for (int r = 0; r < R; ++r) sums[wave][p][r][lane] = acc[p][r];
  __syncthreads();
  // Value e of a lane's fragments: token i16, rows R (4 G + e) .. + R - 1 of a part; a wave each.
  for (int i = wave; i < 4 * P; i += W) {
    const int p = i / 4, e = i % 4, n = n0 + 16 * R * p + R * (4 * G + e);
    float s[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      s[r] = sums[0][p][r][lane][e];
#pragma unroll
      for (int u = 1; u < W; ++u) s[r] += sums[u][p][r][lane][e];
    }
    if (token >= g.m || n >= g.n) continue;
    typedef T row __attribute__((ext_vector_type(R)));
    typedef T anywhere __attribute__((ext_vector_type(R), aligned(sizeof(T))));
    row o;
#pragma unroll
    for (int r = 0; r < R; ++r) o[r] = (T)(s[r] + (g.bias ? g.bias[min(n + r, g.n - 1)] : 0.f));
    T* y = reinterpret_cast<T*>(g.y) + (int64_t)token * g.n + n;
    if (n + R <= g.n) {
      *reinterpret_cast<anywhere*>(y) = o;
    } else {
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (n + r < g.n) y[r] = o[r];
    }
  }
}

// Few fragments take the most workgroups, many the most rows each: x is read and quantized once for
// them, with R = 4 a lane's four scale bytes are one load, and up to 1024 fragments 64 rows each, past
// them 128 are at most one round of the GPU. us in calls from Python (7 at least), R P W = 1 1 8 /
// 2 1 4 / 4 1 4 / 4 2 4 / 4 4 2, a row of bfloat16: 4096 x 4096 6.9 / 7.3 / 9.7 / 13.3 / 26, 4096 x 14336 11.3 / 16.7 /
// 25.3, 8192 x 4096 8.0 / 7.7 / 10.0 / 13.6, 14336 x 4096 12.5 / 11.2 / 10.4 / 14.0, 20480 x 4096 15.6 / 14.9 / 16.0 /
// 14.6 / 27 (16 rows 29 / 21.7 / 20.6 / 17.2 / 29), 128256 x 4096 77 / 62 / 54 / 51.4 / 53.7 (16 rows 164 / 101 /
// 76 / 65 / 58). float32, whose values take twice the registers: 14336 x 4096 - / 13.3 / 11.0 / 15.8, 65536 x
// 4096 - / 41 / 39 / 32 / 30 (16 rows 99 / 62 / 45 / 36), 128256 x 4096 163 / 76 / 75 / 62 / 55 (16 rows 356 / 188 / 119 /
// 88 / 66). The number of x's rows is not asked, so that a row's sums do not depend on the rows beside it.
template <typename T, int R, int P, int W, bool WHOLE>
void launch_few(const FewArgs& g, int fragments, hipStream_t stream) {
  hipLaunchKernelGGL((float4_few_kernel<T, R, P, W, WHOLE>),
                     dim3((unsigned)ceil_div(fragments, R * P), (unsigned)ceil_div(g.m, 16)), dim3(W * 64), 0, stream, g);
}
template <typename T, bool WHOLE>
int launch_few(const FewArgs& g, hipStream_t stream) {
  constexpr bool kLong = sizeof(T) == 4;  // float32 alone comes in the widest form
  const int fragments = (g.n + 15) / 16;
  if (fragments < 320) launch_few<T, 1, 1, 8, WHOLE>(g, fragments, stream);
  else if (fragments <= 640) launch_few<T, 2, 1, 4, WHOLE>(g, fragments, stream);
  else if (fragments <= 1024) launch_few<T, 4, 1, 4, WHOLE>(g, fragments, stream);
  else if (!kLong || fragments < 4096) launch_few<T, 4, 2, 4, WHOLE>(g, fragments, stream);
  else if constexpr (kLong) launch_few<T, 4, 4, 2, WHOLE>(g, fragments, stream);
  return check_launch("float4_few");
}

// WHOLE: the depth is a multiple of 256, so that no block needs its columns counted.
template <typename T>
int launch_few(const FewArgs& g, hipStream_t stream) {
  return g.k % kDepth4 ? launch_few<T, false>(g, stream) : launch_few<T, true>(g, stream);
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

Matrix4 codes_in(Parts& p, int64_t rows, int64_t cols) {
  Matrix4 q{nullptr, nullptr, rows, round_up(cols, kDepth4), round_up(rows, 16)};
  q.data = p.take((size_t)(rows * q.depth / 2));
  q.scale = p.take((size_t)(q.depth / kBlock4 * q.scale_ld));
  return q;
}

struct Saved {
  Matrix4 wt{}, xt{};
  Saved(Parts& p, int64_t m, int64_t n, int64_t k, bool need_x, bool need_w) {
    if (need_x) wt = codes_in(p, k, n);
    if (need_w) xt = codes_in(p, k, m);
  }
};

struct Forward {
  Matrix4 x, w;
  size_t product_bytes;
  void* product;
  Forward(Parts& p, int64_t m, int64_t n, int64_t k) {
    x = codes_in(p, m, k);
    w = codes_in(p, n, k);
    product_bytes = dionw_float4_gemm_workspace(m, n, x.depth);
    product = p.take(product_bytes);
  }
};

struct Backward {
  Matrix4 rows{}, cols{};  // dy by rows and columns
  float* sums = nullptr;
  size_t product_bytes = 0;
  void* product;
  Backward(Parts& p, int64_t m, int64_t n, int64_t k, bool need_x, bool need_w, bool need_b) {
    if (need_x) {
      rows = codes_in(p, m, n);
      product_bytes = dionw_float4_gemm_workspace(m, k, rows.depth);
    }
    if (need_w) {
      cols = codes_in(p, n, m);
      const size_t bytes = dionw_float4_gemm_workspace(n, k, cols.depth);
      if (bytes > product_bytes) product_bytes = bytes;
    }
    if (need_b) sums = static_cast<float*>(p.take((size_t)(ceil_div(m, kTile4) * n) * 4));
    product = p.take(product_bytes);
  }
};

int product(const Matrix4& a, const Matrix4& b, const float* bias, int32_t elem, void* c, void* space,
            size_t bytes, hipStream_t stream) {
  return dionw_float4_gemm(a.rows, b.rows, a.depth, a.data, a.scale, a.scale_ld, b.data, b.scale, b.scale_ld,
                           bias, elem, c, b.rows, space, bytes, stream);
}

// Whether rows of that many columns are ones that the products take.
bool fits_row(int64_t cols) { return cols < 2 * kRowBytes - kDepth4; }

bool good_elem(int32_t e) { return e == kF16 || e == kBF16 || e == kF32; }

}  // namespace
}  // namespace dionw

using namespace dionw;

extern "C" {

void dionw_float4_linear_sizes(int64_t m, int64_t n, int64_t k, int32_t need_x, int32_t need_w,
                               int32_t need_b, size_t* sizes) {
  Parts saved{nullptr}, forward{nullptr}, backward{nullptr};
  Saved s(saved, m, n, k, need_x, need_w);
  Forward f(forward, m, n, k);
  Backward b(backward, m, n, k, need_x, need_w, need_b);
  sizes[0] = saved.used;
  sizes[1] = forward.used;
  sizes[2] = backward.used;
}

int dionw_float4_linear_forward(int32_t x_elem, const void* x, int64_t x_ld, int32_t w_elem,
                                const void* w, int64_t w_ld, const float* bias, int64_t m,
                                int64_t n, int64_t k, int32_t need_x, int32_t need_w, void* y,
                                void* saved, void* scratch, size_t scratch_bytes,
                                hipStream_t stream) {
  DIONW_REQUIRE(good_elem(x_elem) && good_elem(w_elem), "float4_linear: bad element type");
  DIONW_REQUIRE(m >= 0 && n >= 0 && k >= 0, "float4_linear: negative extent");
  DIONW_REQUIRE(saved || !(need_x || need_w) || n == 0 || k == 0, "float4_linear: no room to save");
  // The gradients sum over n and m: refused here rather than after the forward pass.
  DIONW_REQUIRE(fits_row(k) && (!need_x || fits_row(n)) && (!need_w || fits_row(m)),
                "float4_linear: the products take rows of less than 8 MB");
  DIONW_REQUIRE(aligned16(saved) && aligned16(scratch), "float4_linear: buffers need 16-byte alignment");
  Parts kept{static_cast<uint8_t*>(saved)}, room{static_cast<uint8_t*>(scratch)};
  Saved s(kept, m, n, k, need_x, need_w);
  Forward f(room, m, n, k);
  DIONW_REQUIRE(room.used <= scratch_bytes && (scratch || room.used == 0), "float4_linear: scratch too small");
  DIONW_TRY(quantize4_pair({x_elem, x, m, k, x_ld, f.x, s.xt, nullptr},
                           {w_elem, w, n, k, w_ld, f.w, s.wt, nullptr}, stream));
  return product(f.x, f.w, bias, x_elem, y, f.product, f.product_bytes, stream);
}

int dionw_float4_linear_backward(int32_t x_elem, const void* dy, int64_t dy_ld, int32_t w_elem,
                                 int64_t m, int64_t n, int64_t k, int32_t need_x, int32_t need_w,
                                 int64_t seed, const int64_t* seed_at, const void* saved, void* dx,
                                 void* dw, int32_t bias_elem, void* db, void* scratch,
                                 size_t scratch_bytes, hipStream_t stream) {
  DIONW_REQUIRE(good_elem(x_elem) && good_elem(w_elem), "float4_linear: bad element type");
  DIONW_REQUIRE(m >= 0 && n >= 0 && k >= 0, "float4_linear: negative extent");
  DIONW_REQUIRE(aligned16(saved) && aligned16(scratch), "float4_linear: buffers need 16-byte alignment");
  Parts kept{static_cast<uint8_t*>(const_cast<void*>(saved))}, room{static_cast<uint8_t*>(scratch)};
  Saved s(kept, m, n, k, need_x, need_w);
  Backward b(room, m, n, k, need_x, need_w, db != nullptr);
  DIONW_REQUIRE(room.used <= scratch_bytes && (scratch || room.used == 0), "float4_linear: scratch too small");
  DIONW_REQUIRE(saved || kept.used == 0, "float4_linear: nothing was saved");
  const Noise noise{seed, seed_at};
  if (need_x || need_w || db)
    DIONW_TRY(quantize4({x_elem, dy, m, n, dy_ld, b.rows, b.cols, b.sums}, false, &noise, stream));
  if (need_x)
    DIONW_TRY(product(b.rows, s.wt, nullptr, x_elem, dx, b.product, b.product_bytes, stream));
  if (need_w)
    DIONW_TRY(product(b.cols, s.xt, nullptr, w_elem, dw, b.product, b.product_bytes, stream));
  return db ? dionw_sum_parts(b.sums, ceil_div(m, kTile4), n, bias_elem, db, stream) : kOk;
}

size_t dionw_float4_linear_kept_scratch(int64_t m, int64_t n, int64_t k) {
  if (few_rows(m, k)) return 0;
  Parts room{nullptr};
  const Matrix4 x = codes_in(room, m, k);
  room.take(dionw_float4_gemm_workspace(m, n, x.depth));
  return room.used;
}

int dionw_float4_linear_kept(int32_t x_elem, const void* x, int64_t x_ld, const void* w,
                             const void* w_scale, int64_t w_scale_ld, const float* bias, int64_t m,
                             int64_t n, int64_t k, void* y, void* scratch, size_t scratch_bytes,
                             hipStream_t stream) {
  DIONW_REQUIRE(good_elem(x_elem), "float4_linear: bad element type %d", x_elem);
  DIONW_REQUIRE(m >= 0 && n >= 0 && k >= 0 && n < INT32_MAX / 2, "float4_linear: bad extents");
  if (m == 0 || n == 0) return kOk;
  const int64_t depth = round_up(k, kDepth4);
  DIONW_REQUIRE(y && (k == 0 || (x && w && w_scale)), "float4_linear: null pointer");
  DIONW_REQUIRE(x_ld >= k && aligned16(w) && w_scale_ld >= n && w_scale_ld % 16 == 0 && aligned16(w_scale) &&
                    aligned16(scratch),
                "float4_linear: an operand is too small or not aligned");
  if (few_rows(m, k)) {
    DIONW_REQUIRE(depth / kDepth4 < INT32_MAX / 16, "float4_linear: depth too large");
    const FewArgs g{x, x_ld, static_cast<const uint8_t*>(w), static_cast<const uint8_t*>(w_scale),
                    w_scale_ld, bias, y, k, (int32_t)m, (int32_t)n, (int32_t)(depth / kDepth4)};
    if (x_elem == kF16) return launch_few<_Float16>(g, stream);
    if (x_elem == kBF16) return launch_few<__bf16>(g, stream);
    return launch_few<float>(g, stream);
  }
  Parts room{static_cast<uint8_t*>(scratch)};
  const Matrix4 rows = codes_in(room, m, k);
  const size_t bytes = dionw_float4_gemm_workspace(m, n, depth);
  void* space = room.take(bytes);
  DIONW_REQUIRE(room.used <= scratch_bytes && (scratch || room.used == 0), "float4_linear: scratch too small");
  DIONW_TRY(quantize4({x_elem, x, m, k, x_ld, rows, {}, nullptr}, false, nullptr, stream));
  const Matrix4 weight{const_cast<void*>(w), const_cast<void*>(w_scale), n, depth, w_scale_ld};
  return product(rows, weight, bias, x_elem, y, space, bytes, stream);
}

}  // extern "C"

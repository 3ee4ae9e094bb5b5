// The linear layer on 4-bit operands: its passes in order, with their scratch laid out here, and
// the product of a few rows with a kept weight.
#include "float4.h"

#include <type_traits>

namespace dionw {
namespace {

// ---- a few rows ----------------------------------------------------------------------
//
// y = x W^T + b for up to 16 rows of x (the tokens being decoded): every byte of W passes once, from
// memory to registers, and x is quantized on the way, so that the call is one launch. A workgroup takes
// 16 R P rows of W; its waves take the stages of 256 columns in turn and add their sums through LDS, in a
// fixed order. Of a stage, a lane holds one token's (or weight row's) two blocks of 32, number G = lane / 16
// and 4 + G: a block's scale and codes of W are its lane's own, as they lie in memory. x is read two rows a load and
// its codes change lanes through LDS (read as they are needed, 128 bytes a lane apart, 8 rows took 25.6 us
// where now 15.9: 4096 x 14336, float32). A wave reads the next rows while it multiplies the last ones.
// Bound: HBM, n k (1 / 2 + 1 / 32) bytes of W: 128256 x 4096 50.1 us, 5.6 TB/s (reading the codes alone, in
// this order, 45, from end to end 39); the smallest calls: launch and the latency of two dependent reads.
constexpr int kFewFragments = 320, kManyFragments = 1024;  // of 16 rows of W, where the kernel's form changes
int fragments_of(int64_t n) { return (int)((n + 15) / 16); }
// Past 8 rows a deep x costs the kernel as much as W: from some depth on, quantizing first and the product on
// tiles is faster. That depth is 10000 where every workgroup has a CU to itself, less where some wait for a
// second turn. Calls of 16 rows from Python on weights that no cache holds, us, here / there, bfloat16 (float32):
//   4096 rows of W: 4096 columns 7.5 / 11.5, 6144 9.1 / 14.2, 8192 11.1 / 14.2 (13.2 / 14.2), 10240 12.9 / 14.3 (16.3 / 14.3)
//   5104: 2048 7.5 / 11.5, 4096 10.3 / 11.5 (12.9 / 11.5), 6144 14.4 / 14.2
//   8192: 2048 7.5 / 11.5, 4096 11.3 / 11.5 (12.1 / 11.5), 6144 15.5 / 14.3; 16384: 2048 8.3 / 11.5 (9.4 / 11.4), 4096 12.9 /
//   12.0 (16.0 / 12.0)
//   28672: 2048 9.8 / 13.6, 4096 16.4 / 18.8 (17.7 / 19.7), 5120 23.3 / 22.5; 128256: 2048 32 / 36, 4096 61 / 59 (61 / 63).
// 8 rows: 8.9 / 11.2 on 8192 x 4096, 11.0 / 12.0 on 14336 x 4096, 12.8 / 14.7 on 4096 x 14336, 33 / 34 on 16384 x 14336.
bool few_rows(int64_t m, int64_t n, int64_t k) {
  const int fragments = fragments_of(n);
  const bool middle = fragments >= kFewFragments && fragments <= kManyFragments;
  const int64_t deepest = fragments <= 256 ? 8192 : middle ? 2048 : 4096;
  return k > 0 && (m <= 8 || (m <= 16 && k <= deepest));
}

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

// The float32 bits of the largest magnitude of a Square's row.
template <typename T>
__device__ __forceinline__ uint32_t most_of(const Square<T>& v, int i) {
  uint32_t m = 0;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int k = 0; k < 8; ++k) m = max(m, v.w[i][k] & 0x7FFFFFFFu);
    return m;
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) m = Square<T>::larger(m, v.w[i][k] & 0x7FFF7FFFu);
    return Pair<T>::bits(max(m & 0xFFFFu, m >> 16));
  }
}

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
  // A wave's stage of x: codes, at a pitch that spreads 16 rows' reads over the banks, and scales.
  constexpr int kPitch = 36;
  __shared__ __attribute__((aligned(16))) uint32_t x_codes[W][16][kPitch];
  __shared__ uint8_t x_bytes[W][16][8];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int G = lane >> 4, i16 = lane & 15;
  const int n0 = blockIdx.x * 16 * R * P, rows = g.m;
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
  // x as it comes, two rows a load: a lane holds 8 columns of row 2 j + lane / 32.
  const int upper = lane >> 5, eight = lane & 31;
  const T* x = reinterpret_cast<const T*>(g.x) + 8 * eight;
  Square<T> v;
  auto read_x = [&](int kt) {
    const int64_t at = (int64_t)kt * kDepth4, left = g.k - at - 8 * eight;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (2 * j >= rows) break;
      const T* from = x + at + (2 * j + (2 * j + 1 < rows ? upper : 0)) * g.x_ld;
      if (WHOLE || left >= 8) v.load(j, from);
      else v.load(j, from, left);
    }
  };
  // Its codes and scales, a lane's own two blocks of row i16: through LDS, in the wave's own part, so that
  // no one is waited for. Rows past the last are whatever lies there: their sums are not stored.
  i32x4 c[2];
  uint32_t byte[2];
  auto quantize = [&] {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (2 * j >= rows) break;
      const uint32_t b = scale_byte4<false>(largest_of_four(most_of(v, j)));
      x_codes[wave][2 * j + upper][eight] = Codes<T>::row(v, j, power(b));
      if (eight % 4 == 0) x_bytes[wave][2 * j + upper][eight / 4] = (uint8_t)b;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      c[h] = *reinterpret_cast<const i32x4*>(&x_codes[wave][i16][4 * (4 * h + G)]);
      byte[h] = x_bytes[wave][i16][4 * h + G];
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
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
      quantize();
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
    if (i16 >= rows || n >= g.n) continue;
    typedef T row __attribute__((ext_vector_type(R)));
    typedef T anywhere __attribute__((ext_vector_type(R), aligned(sizeof(T))));
    row o;
#pragma unroll
    for (int r = 0; r < R; ++r) o[r] = (T)(s[r] + (g.bias ? g.bias[min(n + r, g.n - 1)] : 0.f));
    T* y = reinterpret_cast<T*>(g.y) + (int64_t)i16 * g.n + n;
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
// them, and with R = 4 a lane's four scale bytes are one load. us in calls from Python (7 at least), R P W = 1 1 8 /
// 2 1 4 / 4 1 4 / 4 2 4 / 4 4 2, a row of bfloat16: 4096 x 4096 7.4 / 7.4 / 9.8 / 13.1 / 25.7, 4096 x 14336 9.9 / 16.0 /
// 24 / 41, 8192 x 4096 7.5 / 7.5 / 10.1 / 13.4, 14336 x 4096 11.0 / 9.4 / 10.6 / 13.7, 20480 x 4096 13.4 / 13.2 /
// 15.7 / 14.3 / 27 (8 rows 17.1 / 15.6 / 17.3 / 14.9 / 28.6), 128256 x 4096 64 / 54 / 52.6 / 50.2 / 51.7 (8 rows 87 / 70 / 62 /
// 55.3 / 53.2); float32: 65536 x 4096 48 / 31.5 / 29.4 / 28.3 / 29.2 (8 rows 70 / 44 / 36.8 / 31.8 / 31.8), 128256 x 4096
// 91 / 56 / 53.5 / 55.0 / 53.2 (8 rows 135 / 84 / 70 / 63.6 / 56.2). The choice does not ask for the number of x's rows: of
// those that come here, a row's sums do not depend on the rows beside it. (More of them take the tiles, which sum in an
// order of their own.)
template <typename T, int R, int P, int W, bool WHOLE>
void launch_few(const FewArgs& g, int fragments, hipStream_t stream) {
  hipLaunchKernelGGL((float4_few_kernel<T, R, P, W, WHOLE>),
                     dim3((unsigned)ceil_div(fragments, R * P)), dim3(W * 64), 0, stream, g);
}
template <typename T, bool WHOLE>
int launch_few(const FewArgs& g, hipStream_t stream) {
  constexpr bool kLong = sizeof(T) == 4;  // float32 alone comes in the widest form
  const int fragments = fragments_of(g.n);
  if (fragments < kFewFragments) launch_few<T, 1, 1, 8, WHOLE>(g, fragments, stream);
  else if (fragments <= kManyFragments) launch_few<T, 2, 1, 4, WHOLE>(g, fragments, stream);
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
  DIONW_REQUIRE(saved || !(need_x || need_w) || m == 0 || n == 0 || k == 0, "float4_linear: no room to save");
  // The gradients sum over n and m: refused here rather than after the forward pass.
  DIONW_REQUIRE(fits_row(k) && (!need_x || fits_row(n)) && (!need_w || fits_row(m)),
                "float4_linear: the products take rows of less than 8 MB");
  DIONW_REQUIRE(aligned16(saved) && aligned16(scratch), "float4_linear: buffers need 16-byte alignment");
  Parts kept{static_cast<uint8_t*>(saved)}, room{static_cast<uint8_t*>(scratch)};
  Saved s(kept, m, n, k, need_x, need_w);
  Forward f(room, m, n, k);
  DIONW_REQUIRE(room.used <= scratch_bytes && (scratch || room.used == 0), "float4_linear: scratch too small");
  if (m == 0) return kOk;  // y and dx are empty, dW and db sums of nothing: nothing that is saved is read
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
  if (few_rows(m, n, k)) return 0;
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
  if (few_rows(m, n, k)) {
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

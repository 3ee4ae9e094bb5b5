// C = alpha A B^T + bias on quantized matrices: 8-bit codes with a scale per row and block of
// 128 columns, or the same values expanded to bfloat16.
//
// Which instruction sums a product goes by its output's type:
// - float16 and bfloat16: v_mfma_scale_f32_16x16x128_f8f6f4 on the codes, one block deep,
//   scales included, at twice the 16-bit rate. It adds groups of 8 products after cutting each
//   to 13 bits below the exponent of the group's largest (measured: beside 2^16, 2^3 counts and
//   2^2 does not), and adds the groups in float32. On normal random operands the result is
//   1.3e-5 off (2-norm), on log-normal ones 6e-5: below the output's rounding (2e-4, 2e-3). Where
//   large products cancel more is lost, up to 7 x 2^-13 of each group's largest product; whoever
//   needs those sums asks for a float32 output.
// - float32: v_mfma_f32_16x16x32_bf16 on codes expanded to bfloat16, scale included, which is
//   exact: 3e-8 off, the accumulation's own rounding. Weight gradients and whatever else asks
//   for float32 sums get them.
#include "product_tiles.h"

using namespace dionw;

extern "C" {

int dionw_float8_gemm_plan(int32_t expanded, int64_t m, int64_t n, int64_t depth, int32_t* side,
                           int32_t* ranges) {
  DIONW_REQUIRE(m > 0 && n > 0 && depth > 0 && depth % kTile == 0 && side && ranges,
                "float8_gemm_plan: bad arguments");
  const Plan p = plan(kCost8, m, n, depth / kTile * (expanded ? 2 : 1));
  *side = kSide[p.tile];
  *ranges = p.splits;
  return kOk;
}

size_t dionw_float8_gemm_workspace(int32_t expanded, int64_t m, int64_t n, int64_t depth) {
  if (m <= 0 || n <= 0 || depth <= 0 || depth % kTile) return 0;
  const Plan p = plan(kCost8, m, n, depth / kTile * (expanded ? 2 : 1));
  return p.splits > 1 ? (size_t)p.splits * m * n * sizeof(float) : 0;
}

int dionw_float8_gemm(int32_t expanded, int64_t m, int64_t n, int64_t depth, const void* a,
                      int64_t lda, const void* a_scale, int64_t a_scale_ld, const void* b,
                      int64_t ldb, const void* b_scale, int64_t b_scale_ld, const float* bias,
                      int32_t elem, void* c, int64_t ldc, void* workspace, size_t workspace_bytes,
                      hipStream_t stream) {
  DIONW_REQUIRE(m >= 0 && n >= 0 && depth >= 0 && depth % kTile == 0 && m < INT32_MAX / 2 &&
                    n < INT32_MAX / 2,
                "float8_gemm: bad extents %lld x %lld x %lld", (long long)m, (long long)n,
                (long long)depth);
  DIONW_REQUIRE(expanded ? elem == kF32 : elem == kF16 || elem == kBF16,
                "float8_gemm: codes give float16 or bfloat16, expanded operands float32");
  if (m == 0 || n == 0) return kOk;
  DIONW_REQUIRE(c && ldc >= n, "float8_gemm: bad output");
  const int64_t size = expanded ? 2 : 1, row = depth * size;
  // A tile's rows are addressed with 32-bit offsets from its first one.
  DIONW_REQUIRE(lda >= depth && ldb >= depth && lda * size < kRowBytes && ldb * size < kRowBytes,
                "float8_gemm: operands need rows of at least their depth, of less than 8 MB");
  DIONW_REQUIRE(lda * size % 16 == 0 && ldb * size % 16 == 0 && aligned16(a) && aligned16(b),
                "float8_gemm: operands need rows at multiples of 16 bytes");
  DIONW_REQUIRE(depth == 0 || (a && b), "float8_gemm: null operand");
  auto scaled = [](const void* s, int64_t ld, int64_t rows) {
    return s && ld >= rows && ld % 16 == 0 && (reinterpret_cast<uintptr_t>(s) & 3) == 0;
  };
  DIONW_REQUIRE(expanded || depth == 0 || (scaled(a_scale, a_scale_ld, m) && scaled(b_scale, b_scale_ld, n)),
                "float8_gemm: codes need a scale for each row, at a pitch that is a multiple of 16");
  DIONW_REQUIRE(expanded || std::max(a_scale_ld, b_scale_ld) <= UINT32_MAX / std::max<int64_t>(row / 128, 1),
                "float8_gemm: a matrix's scales need to lie within 4 GB");
  const Plan p = depth ? plan(kCost8, m, n, row / 128) : Plan{kSmall, 1, 1};
  DIONW_REQUIRE(p.splits == 1 ||
                    (workspace && workspace_bytes >= (size_t)p.splits * m * n * sizeof(float) &&
                     (reinterpret_cast<uintptr_t>(workspace) & 3) == 0),
                "float8_gemm: workspace too small");
  ProductArgs g{};
  g.a = static_cast<const uint8_t*>(a);
  g.lda = lda * size;
  g.a_scale = static_cast<const uint8_t*>(a_scale);
  g.a_scale_ld = a_scale_ld;
  g.b = static_cast<const uint8_t*>(b);
  g.ldb = ldb * size;
  g.b_scale = static_cast<const uint8_t*>(b_scale);
  g.b_scale_ld = b_scale_ld;
  g.bias = bias;
  g.c = c;
  g.ldc = ldc;
  g.m = (int32_t)m;
  g.n = (int32_t)n;
  g.stages = (int32_t)(row / 128);
  g.alpha = expanded ? kExpanded : 1.f;
  float* parts = static_cast<float*>(workspace);
  if (elem == kF16) return launch_product<Form::kCodes8, _Float16>(g, p, parts, stream);
  if (elem == kBF16) return launch_product<Form::kCodes8, __bf16>(g, p, parts, stream);
  return launch_product<Form::kExpanded, float>(g, p, parts, stream);
}

}  // extern "C"

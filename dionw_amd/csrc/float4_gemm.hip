// C = A B^T + bias on 4-bit matrices: v_mfma_scale_f32_16x16x128_f8f6f4 on the codes, scales
// included. A product of two codes is a multiple of 0.25 of at most 36, so that the groups that the
// instruction adds are exact, and the groups are added in float32 (measured on random codes with
// scales of 2^-16 to 2^16: 2e-7 to 4e-7 off after 32768 columns, a third of a serial float32 sum's
// error): every output type is served by it.
#include "product_tiles.h"

#include "float4.h"

using namespace dionw;

extern "C" {

int dionw_float4_gemm_plan(int64_t m, int64_t n, int64_t depth, int32_t* side, int32_t* ranges) {
  DIONW_REQUIRE(m > 0 && n > 0 && depth > 0 && depth % kDepth4 == 0 && side && ranges,
                "float4_gemm_plan: bad arguments");
  const Plan p = plan(kCost4, m, n, depth / kDepth4);
  *side = kSide[p.tile];
  *ranges = p.splits;
  return kOk;
}

size_t dionw_float4_gemm_workspace(int64_t m, int64_t n, int64_t depth) {
  if (m <= 0 || n <= 0 || depth <= 0 || depth % kDepth4) return 0;
  const Plan p = plan(kCost4, m, n, depth / kDepth4);
  return p.splits > 1 ? (size_t)p.splits * m * n * sizeof(float) : 0;
}

int dionw_float4_gemm(int64_t m, int64_t n, int64_t depth, const void* a, const void* a_scale,
                      int64_t a_scale_ld, const void* b, const void* b_scale, int64_t b_scale_ld,
                      const float* bias, int32_t elem, void* c, int64_t ldc, void* workspace,
                      size_t workspace_bytes, hipStream_t stream) {
  DIONW_REQUIRE(m >= 0 && n >= 0 && depth >= 0 && depth % kDepth4 == 0 && m < INT32_MAX / 2 &&
                    n < INT32_MAX / 2,
                "float4_gemm: bad extents %lld x %lld x %lld", (long long)m, (long long)n, (long long)depth);
  DIONW_REQUIRE(elem == kF16 || elem == kBF16 || elem == kF32, "float4_gemm: bad element type %d", elem);
  if (m == 0 || n == 0) return kOk;
  DIONW_REQUIRE(c && ldc >= n, "float4_gemm: bad output");
  // A tile's rows are addressed with 32-bit offsets from its first one.
  DIONW_REQUIRE(depth / 2 < kRowBytes, "float4_gemm: operands need rows of less than 8 MB");
  auto scaled = [](const void* s, int64_t ld, int64_t rows) {
    return s && ld >= rows && ld % 16 == 0 && aligned16(s);
  };
  DIONW_REQUIRE(depth == 0 || (a && b && aligned16(a) && aligned16(b) && scaled(a_scale, a_scale_ld, m) &&
                               scaled(b_scale, b_scale_ld, n)),
                "float4_gemm: operands need codes and a scale for each row at a pitch that is a multiple of "
                "16, at multiples of 16 bytes");
  DIONW_REQUIRE(std::max(a_scale_ld, b_scale_ld) <= UINT32_MAX / std::max<int64_t>(depth / kBlock4, 1),
                "float4_gemm: a matrix's scales need to lie within 4 GB");
  const Plan p = depth ? plan(kCost4, m, n, depth / kDepth4) : Plan{kSmall, 1, 1};
  DIONW_REQUIRE(p.splits == 1 || (workspace && workspace_bytes >= (size_t)p.splits * m * n * sizeof(float) &&
                                  (reinterpret_cast<uintptr_t>(workspace) & 3) == 0),
                "float4_gemm: workspace too small");
  ProductArgs g{};
  g.a = static_cast<const uint8_t*>(a);
  g.lda = depth / 2;
  g.a_scale = static_cast<const uint8_t*>(a_scale);
  g.a_scale_ld = a_scale_ld;
  g.b = static_cast<const uint8_t*>(b);
  g.ldb = depth / 2;
  g.b_scale = static_cast<const uint8_t*>(b_scale);
  g.b_scale_ld = b_scale_ld;
  g.bias = bias;
  g.c = c;
  g.ldc = ldc;
  g.m = (int32_t)m;
  g.n = (int32_t)n;
  g.stages = (int32_t)(depth / kDepth4);
  g.alpha = 1.f;
  float* parts = static_cast<float*>(workspace);
  if (elem == kF16) return launch_product<Form::kCodes4, _Float16>(g, p, parts, stream);
  if (elem == kBF16) return launch_product<Form::kCodes4, __bf16>(g, p, parts, stream);
  return launch_product<Form::kCodes4, float>(g, p, parts, stream);
}

}  // extern "C"

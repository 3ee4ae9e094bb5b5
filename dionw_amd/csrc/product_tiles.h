// The tiles that products of quantized matrices run on, and how a product picks among them:
// C = alpha A B^T + bias, of 8-bit codes with a scale per row and block of 128 columns, of 4-bit codes
// with one per 32, or of the former's values expanded to bfloat16. All of them move 128 bytes of a row
// per stage, so that one tile serves them.
//
// Rows are dealt to fragments so that a lane's scales and outputs lie side by side: of the 16 F
// rows of a wave's F fragments, fragment f's lane i holds row F i + f. Then the F scale bytes
// of a lane are one LDS read, the instruction picks its byte (op_sel), and with the column
// operand first a lane ends with 8 consecutive columns of a row, which it stores at once.
#pragma once

#include "float8.h"

#include <algorithm>
#include <mutex>
#include <type_traits>

namespace dionw {
namespace {

typedef __attribute__((address_space(3))) void* lds_ptr_t;

// What a product's operands hold; 128 bytes of a row are one stage of it.
enum class Form {
  kExpanded,  // 64 columns in bfloat16
  kCodes8,    // 128 columns in 8 bits, with one scale
  kCodes4,    // 256 columns in 4 bits, with 8
};
// A stage's scales of a row, and the words of scale bytes that a lane's fragments of one half take:
// a 4-bit stage is two instructions deep, each of them with a scale for every 32 columns.
template <Form FORM>
constexpr int kScales = FORM == Form::kCodes4 ? 8 : FORM == Form::kCodes8 ? 1 : 0;
template <Form FORM>
constexpr int kWords = FORM == Form::kCodes4 ? 2 : 1;
// LDS bytes of a stage's scales of one operand, as whole loads of a wave fill them.
template <Form FORM, int SIDE>
constexpr int kScaleBytes = FORM == Form::kCodes4 ? (SIDE < 128 ? 1024 : 8 * SIDE) : 256;

struct ProductArgs {
  const uint8_t* a;        // rows of `stages` x 128 bytes at a pitch of lda bytes
  int64_t lda;
  const uint8_t* a_scale;  // codes: [stages x scales][a_scale_ld] exponent bytes
  int64_t a_scale_ld;
  const uint8_t* b;
  int64_t ldb;
  const uint8_t* b_scale;
  int64_t b_scale_ld;
  const float* bias;
  void* c;
  int64_t ldc;
  int64_t split_step;      // elements of C between the sums of two stage ranges
  int32_t m, n;
  int32_t stages, per_split;
  int32_t tiles_m, tiles_n;
  int32_t xcd_group;
  float alpha;
};

// s_waitcnt vmcnt(N) lgkmcnt(R): N loads and the last R LDS reads may be in flight.
template <int N, int R>
__device__ __forceinline__ void wait_vm() {
  __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (R << 8) | ((N >> 4) << 14));
}

// Logical tile of workgroup b: the hardware deals workgroup b to XCD b % 8. group == 0: each
// XCD takes one contiguous range of tiles, so that its L2 sees their shared rows; group > 0:
// runs of `group` tiles in turn (large products, whose operands stream through the Infinity
// Cache), what is left past the last whole turn contiguously. -1 where b only pads the grid
// to a multiple of 8.
__device__ __forceinline__ int xcd_tile(int b, int total, int group) {
  const int x = b % 8, i = b / 8;
  int full = 0;
  if (group > 0) {
    full = total / (8 * group) * (8 * group);
    if (i < full / 8) return ((i / group) * 8 + x) * group + i % group;
  }
  const int rest = total - full, i2 = i - full / 8;
  const int per = rest / 8, extra = rest % 8;
  if (i2 >= per + (x < extra ? 1 : 0)) return -1;
  return full + x * per + min(x, extra) + i2;
}

// The row of a wave's 16 F that slot s (fragment s / 16, lane s % 16) holds.
template <int F>
__device__ __forceinline__ int dealt(int s) {
  return s / (16 * F) * (16 * F) + F * (s % 16) + s % (16 * F) / 16;
}

__device__ __forceinline__ void tile_place(const ProductArgs& g, int t, int& tm, int& tn) {
  const int group = 8 * g.tiles_n;
  const int first = (t / group) * 8;
  const int gm = min(g.tiles_m - first, 8);
  tm = first + (t % group) % gm;
  tn = (t % group) / gm;
}

// One instruction's part of c += b a^T of a fragment pair (4 bits and bfloat16 take two); OA, OB: the
// scales' bytes.
template <Form FORM, int OA, int OB, int P>
__device__ __forceinline__ void multiply_part(i32x8 b, i32x8 a, f32x4& c, const int (&b_scale)[kWords<FORM>],
                                              const int (&a_scale)[kWords<FORM>]) {
  constexpr int W = 4 * P;  // the part's first word of a lane's 8
  if constexpr (FORM == Form::kCodes8) {
    c = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b, a, c, 0, 0, OB, b_scale[0], OA, a_scale[0]);
  } else if constexpr (FORM == Form::kCodes4) {  // the instruction reads 16 bytes of a 4-bit operand
    c = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
        __builtin_shufflevector(b, b, W, W + 1, W + 2, W + 3, -1, -1, -1, -1),
        __builtin_shufflevector(a, a, W, W + 1, W + 2, W + 3, -1, -1, -1, -1), c, 4, 4, OB, b_scale[P], OA,
        a_scale[P]);
  } else {
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
        __builtin_bit_cast(bf16x8, __builtin_shufflevector(b, b, W, W + 1, W + 2, W + 3)),
        __builtin_bit_cast(bf16x8, __builtin_shufflevector(a, a, W, W + 1, W + 2, W + 3)), c, 0, 0, 0);
  }
}

// c0, c1 += b0 a^T, b1 a^T; the scales of b0 and b1 are bytes 0 and 1. A sum's two parts follow each
// other: with the sums taking turns the compiler moves 24 accumulation registers in every two stages of
// the 256 x 256 tile (4 bits, 8192^3: 228 us, in turns 234).
template <Form FORM, int OA>
__device__ __forceinline__ void multiply(i32x8 b0, i32x8 b1, i32x8 a, f32x4& c0, f32x4& c1,
                                         const int (&b_scale)[kWords<FORM>], const int (&a_scale)[kWords<FORM>]) {
  multiply_part<FORM, OA, 0, 0>(b0, a, c0, b_scale, a_scale);
  if constexpr (FORM != Form::kCodes8) multiply_part<FORM, OA, 0, 1>(b0, a, c0, b_scale, a_scale);
  multiply_part<FORM, OA, 1, 0>(b1, a, c1, b_scale, a_scale);
  if constexpr (FORM != Form::kCodes8) multiply_part<FORM, OA, 1, 1>(b1, a, c1, b_scale, a_scale);
}

// A fragment's two chunks of a lane.
__device__ __forceinline__ i32x8 chunks(const unsigned char* lo, const unsigned char* hi) {
  return __builtin_shufflevector(*reinterpret_cast<const i32x4*>(lo),
                                 *reinterpret_cast<const i32x4*>(hi), 0, 1, 2, 3, 4, 5, 6, 7);
}

// A stage's scale bytes of one operand's rows, straight to LDS. Even waves load the first
// operand's and odd ones the second's (several the same bytes), so that every wave issues one
// load. A block's bytes run to a multiple of 16, so a lane's are in bounds; past the last it
// takes the last ones. All of them lie within 2^32 bytes (checked).
// 8 bits: 4 bytes a lane, 256 a load, those past the tile's side repeated. 4 bits: 16 bytes (a chunk
// of 16 rows) a lane; a tile of 256 rows takes two loads. Chunk c of block b lies at place
// c + turn(b) of the block's SIDE / 16: the four blocks that a wave's lanes read together then lie
// in different banks.
template <int SIDE>
__device__ __forceinline__ int turn(int b) {
  return SIDE == 256 ? 4 * (b & 3) : SIDE == 128 ? 2 * (b & 2) : 0;
}
template <Form FORM, int SIDE>
struct ScaleLoad {
#ifdef __HIP_DEVICE_COMPILE__
  __amdgpu_buffer_rsrc_t rsrc;
#endif
  uint32_t off, step;
  int to;  // LDS bytes from the stage's scales on
  __device__ __forceinline__ ScaleLoad(const ProductArgs& g, int wave, int m0, int n0, int first,
                                       int n_stages, int lane) {
#ifdef __HIP_DEVICE_COMPILE__
    const int second = wave & 1;
    const uint8_t* at = second ? g.b_scale : g.a_scale;
    const int64_t ld = second ? g.b_scale_ld : g.a_scale_ld;
    const int row0 = second ? n0 : m0;
    constexpr int S = FORM == Form::kCodes4 ? 8 : 1;
    step = (uint32_t)(S * ld);
    to = second * kScaleBytes<FORM, SIDE>;
    if constexpr (FORM == Form::kCodes4) {
      constexpr int kChunks = SIDE / 16;
      const int part = SIDE == 256 ? wave >> 1 & 1 : 0;
      to += part * 1024;
      const int place = part * 64 + lane, b = place / kChunks % 8;
      const int chunk = (place - turn<SIDE>(b)) & (kChunks - 1);
      off = (uint32_t)(b * ld + min((int64_t)row0 + 16 * chunk, ld - 16));
    } else {
      off = (uint32_t)min((int64_t)row0 + min(4 * lane, SIDE - 4), ld - 4);
    }
    rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)(at + first * (S * ld)), 0, (uint32_t)(n_stages * (S * ld)),
                                             0x00020000);
#endif
  }
  __device__ __forceinline__ void issue(int kt, unsigned char* scales) const {
#ifdef __HIP_DEVICE_COMPILE__
    if constexpr (FORM == Form::kCodes4)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr_t)(scales + to), 16, off, (uint32_t)kt * step, 0, 0);
    else
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr_t)(scales + to), 4, off, (uint32_t)kt * step, 0, 0);
#endif
  }
};

// A row's 8 consecutive columns, from two fragments' accumulators.
template <typename OUT>
struct Row8 {
  typedef OUT type __attribute__((ext_vector_type(8)));
  typedef OUT anywhere __attribute__((ext_vector_type(8), aligned(sizeof(OUT) < 4 ? 2 : 4)));
};
template <typename OUT>
__device__ __forceinline__ typename Row8<OUT>::type row8(f32x4 even, f32x4 odd, float alpha,
                                                         const float (&bias)[8]) {
  typename Row8<OUT>::type o;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    o[2 * e] = (OUT)(alpha * even[e] + bias[2 * e]);
    o[2 * e + 1] = (OUT)(alpha * odd[e] + bias[2 * e + 1]);
  }
  return o;
}

// Stores `left` of a row's 8 columns (8 or more: all).
template <typename OUT>
__device__ __forceinline__ void store_row(OUT* at, typename Row8<OUT>::type o, int left) {
  if (left >= 8) {
    *reinterpret_cast<typename Row8<OUT>::anywhere*>(at) = o;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < left) at[e] = o[e];
  }
}

// The word with the scale bytes of a lane's F fragments: bytes F i16 .. + F - 1 of the wave's 16 F
// rows, at place 8 * scale_shift in the word (shifted down where it is used, not where it is
// read, so that the read is not waited for).
template <int F>
__device__ __forceinline__ uint32_t scale_word(const unsigned char* rows, int i16) {
  return *reinterpret_cast<const uint32_t*>(rows + (F * i16 & ~3));
}
template <Form FORM, int F>
__device__ __forceinline__ int scale_bytes(uint32_t word, int i16) {
  return F == 4 || FORM == Form::kCodes4 ? (int)word : (int)(word >> (16 * (i16 & 1)));
}
// 4-bit codes: the F bytes alone, and their place among a stage's scales of one operand, for the rows
// from `row` on and the first of a lane's two blocks, G (the other, 4 + G, lies 4 SIDE bytes behind it).
template <int F, int SIDE>
__device__ __forceinline__ int scale_place(int row, int G, int i16) {
  const int r = row + F * i16;
  return G * SIDE + ((r / 16 + turn<SIDE>(G)) & (SIDE / 16 - 1)) * 16 + r % 16;
}
template <int F>
__device__ __forceinline__ uint32_t scale_at(const unsigned char* at) {
  if constexpr (F == 4) return *reinterpret_cast<const uint32_t*>(at);
  else return *reinterpret_cast<const uint16_t*>(at);
}

// A lane's 8 columns' bias.
__device__ __forceinline__ void load_bias(const ProductArgs& g, int q, float (&bias)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) bias[e] = 0.f;
  if (g.bias) {
#pragma unroll
    for (int e = 0; e < 8; ++e) bias[e] = g.bias[min(q + e, g.n - 1)];
  }
}

// ---- quadrant tiles ------------------------------------------------------------------
//
// 256 x 256 outputs by 8 waves, one workgroup per CU, and 128 x 128 by 4, two per CU. The
// tile splits into two halves each way; a wave owns FI x FJ fragments of 16 x 16 in each of
// the four quadrants and multiplies them in the order 00, 01, 11, 10: each step changes one
// operand's half, whose fragments are read from LDS under the instructions of the step before.
// An operand's half stage is an LDS slot of its own in a ring of two stages, filled by
// direct-to-LDS loads up to two stages ahead; the workgroup meets at two barriers per stage.
// Every wave issues the same loads, so the counts of the waits are exact: rows past the edge
// load the last row (outputs that are never stored see them). A stage's scale bytes come the
// same way, one load of a wave for 256 rows, and are read a stage ahead. Whole tiles store from
// registers, 64 bytes of 16 rows an instruction.
// Bound: the board's power (8 bits: 8192^3 395 us, 2785 TFLOP/s, 366 sustained at 1387 W of 1400 and 1.8 GHz,
// the matrix pipe 77% busy; 4 bits: 228 us, 4820 TFLOP/s, 237 sustained at 1396 W and 1.7 GHz, 61% busy; on constant
// operands 169 at 1324 W and 2.36 GHz, on zeros 167 at 1164 W, where neither power nor the pipe (66%) is the bound;
// the instruction alone on random registers 7200 TFLOP/s; expanded 14336 x 4096 x 8192 720 us, 1336, at 1400 W and 2.05 GHz, 68%);
// at few stages the first loads and the stores (plan_time; 8192 x 2304 x 768 24 us, 20%). Stores are
// 14% of 4-bit 8192 x 14336 x 4096 (229 us, 197 without them): they wait for memory. Not kept there: stores
// past the caches (241), through LDS in whole rows (232), and workgroups that take one tile after another
// and load the next one's first stages before the stores (278: the sums leave their registers).
template <int WM_, int WN_, int FI_, int FJ_>
struct QuadCfg {
  static constexpr int WM = WM_, WN = WN_, FI = FI_, FJ = FJ_;
  static constexpr int waves = WM * WN, threads = waves * 64;
  static constexpr int HM = WM * FI * 16, HN = WN * FJ * 16;  // half tile rows / columns
  static constexpr int BM = 2 * HM, BN = 2 * HN;
  static constexpr int half = HM * 128;        // bytes of a half stage
  static constexpr int L = half / 16 / threads;  // loads per lane
  template <Form FORM>
  static constexpr size_t lds_bytes = (size_t)8 * half + 4 * kScaleBytes<FORM, BM>;
  static_assert(HM == HN && L >= 1 && FJ == 2, "square tiles, pairs of column fragments");
};

using BigTile = QuadCfg<2, 4, 4, 2>;  // 256x256
using MidTile = QuadCfg<2, 2, 2, 2>;  // 128x128

template <typename CFG, Form FORM, typename OUT>
__device__ __forceinline__ void quad_tile(const ProductArgs& g, int w) {
#ifdef __HIP_DEVICE_COMPILE__  // the host pass has no buffer-resource type
  constexpr int HM = CFG::HM, HN = CFG::HN, FI = CFG::FI, FJ = CFG::FJ, BM = CFG::BM, BN = CFG::BN;
  constexpr int L = CFG::L, W = CFG::waves, S = kScales<FORM> ? 1 : 0;  // S: scale loads of a stage
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  constexpr int SB = kScaleBytes<FORM, BM>;
  // The scales come first, so that a read's offset from a lane's place fits its instruction.
  unsigned char* lds_s = smem;                    // [buffer][operand][SB]
  unsigned char* lds_a = smem + 4 * SB;           // [buffer][half][HM][128]
  unsigned char* lds_b = lds_a + 4 * CFG::half;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / CFG::WN, wn = wave % CFG::WN;
  const int tiles = g.tiles_m * g.tiles_n, split = w / tiles;
  int tm, tn;
  tile_place(g, w - split * tiles, tm, tn);
  const int m0 = tm * BM, n0 = tn * BN;
  const int first = split * g.per_split, n_stages = min(g.per_split, g.stages - first);
  const uint8_t* A = g.a + (int64_t)m0 * g.lda + (int64_t)first * 128;
  const uint8_t* B = g.b + (int64_t)n0 * g.ldb + (int64_t)first * 128;
  // Byte offsets of a lane's 16-byte loads of each half: load j of wave w fills the 1 KB at
  // 1024 (W j + w) of the half, lane i at + 16 i; chunk c of slot row r lies at c ^ (r / 2 % 8),
  // so that the 16 lanes of a read phase touch 16 different 16-byte bank groups.
  uint32_t a_off[2][L], b_off[2][L];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int j = 0; j < L; ++j) {
      const int pos = (j * W + wave) * 64 + lane;
      const int slot = pos >> 3, ch = (pos & 7) ^ ((slot >> 1) & 7);
      a_off[h][j] = (uint32_t)min(h * HM + dealt<FI>(slot), g.m - 1 - m0) * (uint32_t)g.lda + 16 * ch;
      b_off[h][j] = (uint32_t)min(h * HN + dealt<FJ>(slot), g.n - 1 - n0) * (uint32_t)g.ldb + 16 * ch;
    }
  const uint32_t a_bytes = (uint32_t)(min(BM, g.m - m0) - 1) * (uint32_t)g.lda + (uint32_t)n_stages * 128;
  const uint32_t b_bytes = (uint32_t)(min(BN, g.n - n0) - 1) * (uint32_t)g.ldb + (uint32_t)n_stages * 128;
  const auto a_rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)A, 0, a_bytes, 0x00020000);
  const auto b_rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)B, 0, b_bytes, 0x00020000);
  auto load_a = [&](int kt, int buf, int h) {
#pragma unroll
    for (int j = 0; j < L; ++j)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          a_rsrc, (lds_ptr_t)(lds_a + (2 * buf + h) * CFG::half + (j * W + wave) * 1024), 16,
          a_off[h][j], kt * 128, 0, 0);
  };
  auto load_b = [&](int kt, int buf, int h) {
#pragma unroll
    for (int j = 0; j < L; ++j)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          b_rsrc, (lds_ptr_t)(lds_b + (2 * buf + h) * CFG::half + (j * W + wave) * 1024), 16,
          b_off[h][j], kt * 128, 0, 0);
  };
  const ScaleLoad<FORM, BM> scale_load(g, wave, m0, n0, first, n_stages, lane);
  auto load_s = [&](int kt, int buf) {
    if constexpr (S) scale_load.issue(kt, lds_s + buf * 2 * SB);
  };

  // A fragment's lane i holds its row i % 16 and, of the 128 bytes, chunks i / 16 and 4 + i / 16
  // (any order serves that both operands share).
  const int G = lane >> 4, i16 = lane & 15, sw = (i16 >> 1) & 7;
  const unsigned char* a_rd[2];
  const unsigned char* b_rd[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    a_rd[k] = lds_a + (wm * FI * 16 + i16) * 128 + (((4 * k + G) ^ sw) << 4);
    b_rd[k] = lds_b + (wn * FJ * 16 + i16) * 128 + (((4 * k + G) ^ sw) << 4);
  }
  auto read_a = [&](i32x8 (&f)[FI], int i, int buf, int h) {
    const int at = (2 * buf + h) * CFG::half + i * 16 * 128;
    f[i] = chunks(a_rd[0] + at, a_rd[1] + at);
  };
  auto read_b = [&](i32x8 (&f)[FJ], int j, int buf, int h) {
    const int at = (2 * buf + h) * CFG::half + j * 16 * 128;
    f[j] = chunks(b_rd[0] + at, b_rd[1] + at);
  };
  struct Scales {
    uint32_t a[2][kWords<FORM>], b[2][kWords<FORM>];  // by half: the words of scale_word
  };
  const unsigned char *a_scale[2], *b_scale[2];  // 4 bits: the bytes by half
  if constexpr (FORM == Form::kCodes4) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      a_scale[h] = lds_s + scale_place<FI, BM>(h * HM + wm * FI * 16, G, i16);
      b_scale[h] = lds_s + SB + scale_place<FJ, BM>(h * HN + wn * FJ * 16, G, i16);
    }
  }
  auto read_s = [&](Scales& s, int buf) {
    if constexpr (FORM == Form::kCodes4) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int at = buf * 2 * SB + k * 4 * BM;
          s.a[h][k] = scale_at<FI>(a_scale[h] + at);
          s.b[h][k] = scale_at<FJ>(b_scale[h] + at);
        }
    } else if constexpr (S) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        s.a[h][0] = scale_word<FI>(lds_s + buf * 2 * SB + h * HM + wm * FI * 16, i16);
        s.b[h][0] = scale_word<FJ>(lds_s + buf * 2 * SB + SB + h * HN + wn * FJ * 16, i16);
      }
    }
  };

  // Names an accumulation register, so that the compiler keeps the sums in them. Without it the
  // scaled instruction's results wander through the vector registers, and the 256 x 256 tile
  // spills 400 of them.
  int unused;
  asm volatile("" : "=a"(unused));
  f32x4 acc[2 * FI][2 * FJ];
#pragma unroll
  for (int i = 0; i < 2 * FI; ++i)
#pragma unroll
    for (int j = 0; j < 2 * FJ; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][j][e] = 0.f;
  i32x8 a[FI], bx[FJ], by[FJ];
  Scales sx{}, sy{};
#define QUAD_FENCE __builtin_amdgcn_sched_barrier(0);
  // READS: the wave's last LDS reads that may still be on their way when it meets the others;
  // the slots refilled after the sync must not be among theirs.
#define QUAD_SYNC(VM, READS)                                                    \
  QUAD_FENCE                                                                    \
  wait_vm<VM, READS>();                                                         \
  __builtin_amdgcn_s_barrier();                                                 \
  QUAD_FENCE
  auto row = [&](auto qi_, auto qj_, auto i_, i32x8 (&b)[FJ], const int (&s)[2][2][kWords<FORM>]) {
    constexpr int qi = decltype(qi_)::value, qj = decltype(qj_)::value, i = decltype(i_)::value;
    multiply<FORM, i>(b[0], b[1], a[i], acc[qi * FI + i][qj * FJ], acc[qi * FI + i][qj * FJ + 1], s[1][qj], s[0][qi]);
    QUAD_FENCE
  };
  using I0 = std::integral_constant<int, 0>;
  using I1 = std::integral_constant<int, 1>;
  using I2 = std::integral_constant<int, 2>;
  auto rows = [&](auto body) {  // body(i) for every row fragment
    body(I0{});
    body(I1{});
    if constexpr (FI == 4) {
      body(I2{});
      body(std::integral_constant<int, 3>{});
    }
  };
  // One stage. b0 holds B0(kt) and s0 its scales at entry; b1 holds B0(kt + 1) and s1 its scales
  // at exit. tail 0: two more stages follow at least; 1: one; 2: none. Loads are issued in the
  // order S B0 A0 B1 A1 of each stage.
  auto stage = [&](auto buf_, auto tail_, int kt, i32x8 (&b0)[FJ], i32x8 (&b1)[FJ],
                   const Scales& s0, Scales& s1) {
    constexpr int buf = decltype(buf_)::value, tail = decltype(tail_)::value;
    int s[2][2][kWords<FORM>];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int k = 0; k < kWords<FORM>; ++k) {
        s[0][h][k] = scale_bytes<FORM, FI>(s0.a[h][k], i16);
        s[1][h][k] = scale_bytes<FORM, FJ>(s0.b[h][k], i16);
      }
    // rows half 0 x columns half 0; B1(kt) is read. Pending: A0(kt), B1(kt) and A1(kt) have
    // landed. Refilled next: A1(kt - 1), B0(kt), S(kt), all read before A0(kt).
    QUAD_SYNC((tail != 2 ? 3 * L + S : 0), 2 * FI)
    rows([&](auto i) {
      row(I0{}, I0{}, i, b0, s);
      if (i < FJ) read_b(b1, i, buf, 1);
      if (i == 0 && tail != 2) load_a(kt + 1, buf ^ 1, 1);
      QUAD_FENCE
    });
    // 0 x 1; A1(kt) replaces A0(kt)
    rows([&](auto i) {
      row(I0{}, I1{}, i, b1, s);
      read_a(a, i, buf, 1);
      if (i == 0 && tail == 0) {
        load_s(kt + 2, buf);
        load_b(kt + 2, buf, 0);
      }
      QUAD_FENCE
    });
    // 1 x 1; B0(kt + 1) replaces B1(kt). Pending: A1(kt). Refilled next: A0(kt), B1(kt).
    if (tail != 2) {
      QUAD_SYNC((tail == 0 ? 3 * L + S : 2 * L), 2 * FI)
    }
    rows([&](auto i) {
      row(I1{}, I1{}, i, b1, s);
      if (i == 0 && tail == 0) load_a(kt + 2, buf, 0);
      if (tail != 2 && i == 0) read_s(s1, buf ^ 1);
      QUAD_FENCE
    });
    if (tail != 2) {
#pragma unroll
      for (int j = 0; j < FJ; ++j) read_b(b1, j, buf ^ 1, 0);
      QUAD_FENCE
    }
    // 1 x 0; A0(kt + 1) replaces A1(kt)
    rows([&](auto i) {
      row(I1{}, I0{}, i, b0, s);
      if (tail != 2) read_a(a, i, buf ^ 1, 0);
      if (i == 0 && tail == 0) load_b(kt + 2, buf, 1);
      QUAD_FENCE
    });
  };
  auto first_reads = [&](int buf, i32x8 (&b)[FJ], Scales& s) {
    read_s(s, buf);
#pragma unroll
    for (int j = 0; j < FJ; ++j) read_b(b, j, buf, 0);
    QUAD_FENCE
#pragma unroll
    for (int i = 0; i < FI; ++i) read_a(a, i, buf, 0);
  };

  // Stage kt sits in buffer (kt + n_stages) & 1, so that the last two stages always sit in
  // buffers 0 and 1.
  const int p0 = n_stages & 1;
  load_s(0, p0);
  load_b(0, p0, 0);
  load_a(0, p0, 0);
  load_b(0, p0, 1);
  load_a(0, p0, 1);
  load_s(1, p0 ^ 1);
  load_b(1, p0 ^ 1, 0);
  load_a(1, p0 ^ 1, 0);
  load_b(1, p0 ^ 1, 1);
  QUAD_SYNC((5 * L + S), 15)
  int kt = 0;
  if (p0) {
    first_reads(1, by, sy);
    stage(I1{}, I0{}, 0, by, bx, sy, sx);
    kt = 1;
  } else {
    first_reads(0, bx, sx);
  }
  for (; kt < n_stages - 2; kt += 2) {
    stage(I0{}, I0{}, kt, bx, by, sx, sy);
    stage(I1{}, I0{}, kt + 1, by, bx, sy, sx);
  }
  stage(I0{}, I1{}, n_stages - 2, bx, by, sx, sy);
  stage(I1{}, I2{}, n_stages - 1, by, bx, sy, sx);
#undef QUAD_FENCE
#undef QUAD_SYNC
  OUT* C = reinterpret_cast<OUT*>(g.c) + split * g.split_step + m0 * g.ldc + n0;
  const int r0 = wm * FI * 16 + FI * i16, q0 = wn * FJ * 16 + 8 * G;  // a lane's place in a quadrant
  if (m0 + BM <= g.m && n0 + BN <= g.n) {
#pragma unroll
    for (int qj = 0; qj < 2; ++qj) {
      float bias[8];
      load_bias(g, n0 + qj * HN + q0, bias);
#pragma unroll
      for (int qi = 0; qi < 2; ++qi) {
        OUT* at = C + (qi * HM + r0) * g.ldc + qj * HN + q0;
#pragma unroll
        for (int i = 0; i < FI; ++i, at += g.ldc)
          *reinterpret_cast<typename Row8<OUT>::anywhere*>(at) =
              row8<OUT>(acc[qi * FI + i][qj * FJ], acc[qi * FI + i][qj * FJ + 1], g.alpha, bias);
      }
    }
    return;
  }
  // A ragged tile goes through LDS, a quadrant at a time, so that what guards its edges is a loop.
  OUT* quadrant = reinterpret_cast<OUT*>(smem);
  static_assert((size_t)HM * HN * sizeof(OUT) <= CFG::template lds_bytes<FORM>, "a quadrant fits");
#pragma unroll
  for (int qj = 0; qj < 2; ++qj) {
    float bias[8];
    load_bias(g, n0 + qj * HN + q0, bias);
#pragma unroll
    for (int qi = 0; qi < 2; ++qi) {
      __syncthreads();  // the last stage, the quadrant before
#pragma unroll
      for (int i = 0; i < FI; ++i)
        *reinterpret_cast<typename Row8<OUT>::type*>(quadrant + (r0 + i) * HN + q0) =
            row8<OUT>(acc[qi * FI + i][qj * FJ], acc[qi * FI + i][qj * FJ + 1], g.alpha, bias);
      __syncthreads();
      const int rows = min(HM, g.m - m0 - qi * HM), cols = min(HN, g.n - n0 - qj * HN);
#pragma unroll 1
      for (int at = tid; at < HM * HN / 8; at += CFG::threads) {
        const int r = at / (HN / 8), q = at % (HN / 8) * 8;
        if (r < rows && q < cols)
          store_row<OUT>(C + (qi * HM + r) * g.ldc + qj * HN + q,
                         *reinterpret_cast<const typename Row8<OUT>::type*>(quadrant + r * HN + q),
                         cols - q);
      }
    }
  }
#endif
}

// ---- 64 x 64 tiles -------------------------------------------------------------------
//
// 4 waves of 32 x 32 and a ring of 8 stages, 7 of them on their way: for products of so few
// tiles that their time is one tile's chain of stages, and for few rows, where the other
// operand streams from memory and a CU needs about 64 KB on its way to keep up. A stage takes
// 0.28 us, 57 GB/s into each CU's LDS. 64 x 14336 x 4096 13.2 us (128 tiles 18.9), 512^3 4.4 (5.5). Not
// kept: 128 x 64 outputs on 6 stages, 0.39 us a stage.
struct SmallTile {
  static constexpr int threads = 256, BM = 64, BN = 64, ring = 8;
  static constexpr int operand = 64 * 128;
  template <Form FORM>
  static constexpr int slot = 2 * operand + 2 * kScaleBytes<FORM, BM>;  // A, B, their scales
  template <Form FORM>
  static constexpr size_t lds_bytes = (size_t)ring * slot<FORM>;
};

// s_waitcnt for n stages of P loads in flight, n <= 6.
template <int P>
__device__ __forceinline__ void wait_stages(int n) {
  switch (n) {
    case 0: wait_vm<0, 15>(); break;
    case 1: wait_vm<P, 15>(); break;
    case 2: wait_vm<2 * P, 15>(); break;
    case 3: wait_vm<3 * P, 15>(); break;
    case 4: wait_vm<4 * P, 15>(); break;
    case 5: wait_vm<5 * P, 15>(); break;
    default: wait_vm<6 * P, 15>(); break;
  }
}

template <Form FORM, typename OUT>
__device__ __forceinline__ void small_tile(const ProductArgs& g, int w) {
#ifdef __HIP_DEVICE_COMPILE__
  using CFG = SmallTile;
  constexpr int R = CFG::ring, BM = CFG::BM, BN = CFG::BN, P = 4 + (kScales<FORM> ? 1 : 0),
                SB = kScaleBytes<FORM, BM>;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 1, wn = wave & 1;
  const int tiles = g.tiles_m * g.tiles_n, split = w / tiles;
  int tm, tn;
  tile_place(g, w - split * tiles, tm, tn);
  const int m0 = tm * BM, n0 = tn * BN;
  const int first = split * g.per_split, n_stages = min(g.per_split, g.stages - first);
  const uint8_t* A = g.a + (int64_t)m0 * g.lda + (int64_t)first * 128;
  const uint8_t* B = g.b + (int64_t)n0 * g.ldb + (int64_t)first * 128;
  uint32_t a_off[2], b_off[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int pos = (j * 4 + wave) * 64 + lane;
    const int slot = pos >> 3, ch = (pos & 7) ^ ((slot >> 1) & 7);
    a_off[j] = (uint32_t)min(dealt<2>(slot), g.m - 1 - m0) * (uint32_t)g.lda + 16 * ch;
    b_off[j] = (uint32_t)min(dealt<2>(slot), g.n - 1 - n0) * (uint32_t)g.ldb + 16 * ch;
  }
  const uint32_t a_bytes = (uint32_t)(min(BM, g.m - m0) - 1) * (uint32_t)g.lda + (uint32_t)n_stages * 128;
  const uint32_t b_bytes = (uint32_t)(min(BN, g.n - n0) - 1) * (uint32_t)g.ldb + (uint32_t)n_stages * 128;
  const auto a_rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)A, 0, a_bytes, 0x00020000);
  const auto b_rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)B, 0, b_bytes, 0x00020000);
  const ScaleLoad<FORM, BM> scale_load(g, wave, m0, n0, first, n_stages, lane);
  auto issue = [&](int kt) {
    unsigned char* stage = smem + (kt % R) * CFG::template slot<FORM>;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      __builtin_amdgcn_raw_ptr_buffer_load_lds(a_rsrc, (lds_ptr_t)(stage + (j * 4 + wave) * 1024), 16,
                                               a_off[j], kt * 128, 0, 0);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          b_rsrc, (lds_ptr_t)(stage + CFG::operand + (j * 4 + wave) * 1024), 16, b_off[j], kt * 128, 0, 0);
    }
    if constexpr (kScales<FORM>) scale_load.issue(kt, stage + 2 * CFG::operand);
  };
  const int G = lane >> 4, i16 = lane & 15, sw = (i16 >> 1) & 7;
  struct Frags {
    i32x8 a[2], b[2];
    uint32_t as[kWords<FORM>], bs[kWords<FORM>];
  };
  int a_place = 0, b_place = 0;  // 4 bits: the scales' words
  if constexpr (FORM == Form::kCodes4) {
    a_place = scale_place<2, BM>(wm * 32, G, i16);
    b_place = SB + scale_place<2, BM>(wn * 32, G, i16);
  }
  auto read = [&](Frags& f, int kt) {
    const unsigned char* stage = smem + (kt % R) * CFG::template slot<FORM>;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const unsigned char* at = stage + (i * 16 + i16) * 128;
      const unsigned char *ra = at + wm * 32 * 128, *rb = at + CFG::operand + wn * 32 * 128;
      f.a[i] = chunks(ra + ((G ^ sw) << 4), ra + (((4 + G) ^ sw) << 4));
      f.b[i] = chunks(rb + ((G ^ sw) << 4), rb + (((4 + G) ^ sw) << 4));
    }
    const unsigned char* s = stage + 2 * CFG::operand;
    if constexpr (FORM == Form::kCodes4) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        f.as[k] = scale_at<2>(s + k * 4 * BM + a_place);
        f.bs[k] = scale_at<2>(s + k * 4 * BM + b_place);
      }
    } else if constexpr (FORM == Form::kCodes8) {
      f.as[0] = scale_word<2>(s + wm * 32, i16);
      f.bs[0] = scale_word<2>(s + SB + wn * 32, i16);
    } else {
      f.as[0] = f.bs[0] = 0;
    }
  };
  f32x4 acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][j][e] = 0.f;
  // Stage kt is multiplied while stage kt + 1 is read and stage kt - 1 + R requested (into the
  // slot of kt - 1, which every wave has read).
  auto step = [&](auto more_, int kt, Frags& now, Frags& next) {
    if (decltype(more_)::value) {
      __builtin_amdgcn_sched_barrier(0);
      wait_stages<P>(min(R - 3, n_stages - 2 - kt));
      // The reads of stage kt, whose slot is refilled after the next barrier, are complete:
      // what they fill is multiplied below, before that barrier.
      __builtin_amdgcn_s_barrier();
      __builtin_amdgcn_sched_barrier(0);
      read(next, kt + 1);
      if (kt - 1 + R < n_stages) issue(kt - 1 + R);
      __builtin_amdgcn_sched_barrier(0);
    }
    int as[kWords<FORM>], bs[kWords<FORM>];
#pragma unroll
    for (int k = 0; k < kWords<FORM>; ++k) {
      as[k] = scale_bytes<FORM, 2>(now.as[k], i16);
      bs[k] = scale_bytes<FORM, 2>(now.bs[k], i16);
    }
    multiply<FORM, 0>(now.b[0], now.b[1], now.a[0], acc[0][0], acc[0][1], bs, as);
    multiply<FORM, 1>(now.b[0], now.b[1], now.a[1], acc[1][0], acc[1][1], bs, as);
  };
#pragma unroll 1
  for (int s = 0; s < min(R - 1, n_stages); ++s) issue(s);
  wait_stages<P>(min(R - 2, n_stages - 1));
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  Frags x, y;
  read(x, 0);
  int kt = 0;
  for (; kt + 2 < n_stages; kt += 2) {
    step(std::true_type{}, kt, x, y);
    step(std::true_type{}, kt + 1, y, x);
  }
  if (kt + 1 < n_stages) {
    step(std::true_type{}, kt, x, y);
    step(std::false_type{}, kt + 1, y, x);
  } else {
    step(std::false_type{}, kt, x, y);
  }
  const int q = n0 + wn * 32 + 8 * G;
  float bias[8];
  load_bias(g, q, bias);
  const int row0 = m0 + wm * 32 + 2 * i16;
  OUT* at = reinterpret_cast<OUT*>(g.c) + split * g.split_step + row0 * g.ldc + q;
#pragma unroll
  for (int i = 0; i < 2; ++i, at += g.ldc)
    if (row0 + i < g.m && q < g.n)
      store_row<OUT>(at, row8<OUT>(acc[i][0], acc[i][1], g.alpha, bias), g.n - q);
#endif
}

template <typename CFG, Form FORM, typename OUT>
__global__ __launch_bounds__(CFG::threads, 1) __attribute__((amdgpu_waves_per_eu(2, 2))) void
product_kernel(ProductArgs g, int total) {
  const int w = xcd_tile((int)blockIdx.x, total, g.xcd_group);
  if (w < 0) return;  // the whole workgroup: w depends on blockIdx only
  if constexpr (std::is_same<CFG, SmallTile>::value)
    small_tile<FORM, OUT>(g, w);
  else
    quad_tile<CFG, FORM, OUT>(g, w);
}

// C = alpha (the ranges' sums in order) + bias, 4 elements a thread, the loads of 4 ranges at once.
template <typename OUT>
__global__ __launch_bounds__(256) void join_splits_kernel(ProductArgs g, const float* parts, int splits) {
  const int64_t total = (int64_t)g.m * g.n, at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (at >= total) return;
  typedef float f4any __attribute__((ext_vector_type(4), aligned(4)));
  const bool whole = at + 4 <= total;
  const uint32_t left = whole ? 4 : (uint32_t)(total - at);
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  for (int k0 = 0; k0 < splits; k0 += 4) {
    f32x4 v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float* from = parts + min(k0 + k, splits - 1) * total + at;
      if (whole) {
        v[k] = *reinterpret_cast<const f4any*>(from);
      } else {
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) v[k][e] = e < left ? from[e] : 0.f;
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k0 + k < splits) s = k0 + k ? s + v[k] : v[k];
  }
  int64_t row = total <= UINT32_MAX ? (uint32_t)at / (uint32_t)g.n : at / g.n;
  int col = (int)(at - row * g.n);
  OUT* c = reinterpret_cast<OUT*>(g.c);
  if (whole && col + 4 <= g.n) {
    typedef OUT o4 __attribute__((ext_vector_type(4)));
    typedef OUT o4any __attribute__((ext_vector_type(4), aligned(sizeof(OUT))));
    o4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = (OUT)(g.alpha * s[e] + (g.bias ? g.bias[col + e] : 0.f));
    *reinterpret_cast<o4any*>(c + row * g.ldc + col) = o;
    return;
  }
#pragma unroll
  for (uint32_t e = 0; e < 4; ++e) {
    if (e < left) c[row * g.ldc + col] = (OUT)(g.alpha * s[e] + (g.bias ? g.bias[col] : 0.f));
    if (++col == g.n) {
      col = 0;
      ++row;
    }
  }
}

// C = bias, for a depth of zero.
template <typename OUT>
__global__ __launch_bounds__(256) void fill_bias_kernel(ProductArgs g) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= (int64_t)g.m * g.n) return;
  const int64_t row = at / g.n, col = at - row * g.n;
  reinterpret_cast<OUT*>(g.c)[row * g.ldc + col] = (OUT)(g.bias ? g.bias[col] : 0.f);
}

// How a product is launched: its tile and in how many ranges its depth is split.
enum Tile : int { kBig = 0, kMid = 1, kSmall = 2 };
constexpr int kSide[3] = {256, 128, 64};
constexpr int kMinStages[3] = {2, 2, 1};

struct Plan {
  int tile;
  int splits, per_split;
};

// Estimated time, us: rounds of one workgroup per CU, each its stages plus a fixed part (first
// loads, stores; a second round of 64 x 64 tiles waits for the LDS of the first), and, where the
// depth is split, one more launch and the sums' way to memory and back. Measured, us on 256 / 128 / 64
// tiles, the time of an empty launch (3) included:
// 8 bits: 8192^3 395 / 448 / 1338, 8192 x 14336 x 4096 358 / 423 / 1285, 4096^3 56 / 63 / 186;
// 8192 x 2304 x 768 28 / 23 / 71, 3001 x 1408 x 2048 25 / 16 / 35, 2048^3 24 / 11 / 29; 64 x 14336 x
// 4096 39 / 19 / 14, 1024^3 15 / 7.0 / 6.1, 512^3 11 / 5.7 / 4.7. Split in 1 / 2 / 4 / 8, 128 tiles:
// 100 x 4096 x 14336 48 / 32 / 23 / 22, expanded 2304 x 768 x 8192 56 / 41 / 41 / 48.
// 4 bits, whose stages are twice as deep: 8192 x 14336 x 4096 232 / 260, 8192 x 4096 x 14336 192 / 233 /
// 642, 4096^3 35 / 40 / 116, 4096 x 14336 x 4096 128 / 133 / 401, 5000^3 74 / 77 / 214; 8192 x 2304 x 768
// 24 / 17 / 30, 3001 x 1408 x 2048 19 / 13 / 25, 1024 x 4096 x 4096 26 / 13 / 31; 256 x 4096 x 4096 25 / 12 /
// 8.7, 64 x 4096 x 4096 27 / 13 / 8.4. Split: 100 x 4096 x 14336 29 whole on 128 tiles, 16.5 in 7
// there (chosen) and in 2 on 64; 700 x 700 x 16384 24.5 whole on 64 tiles, 18.5 in 2, 19.1 in 6 on 128 (chosen);
// 130 x 770 x 6144 11.2 whole on 64 tiles, 10.2 in 3 (chosen), 9.7 in 4 or 6. Either rule takes the fastest on
// nearly all of them, and on these none that is more than 5% slower.
struct Cost {
  double stage[3], fixed[3];
};
constexpr Cost kCost8{{1.4, 0.42, 0.28}, {5.0, 1.0, 0.6}}, kCost4{{1.56, 0.5, 0.33}, {7.5, 1.4, 0.6}};

inline double plan_time(const Cost& cost, int64_t m, int64_t n, int64_t stages, int tile, int64_t splits) {
  const int64_t per = ceil_div(stages, splits);
  const int64_t rounds = ceil_div(ceil_div(m, kSide[tile]) * ceil_div(n, kSide[tile]) * splits, 256);
  double t = (double)rounds * (cost.stage[tile] * (double)per + cost.fixed[tile] +
                               (tile == kSmall && rounds > 1 ? 1.4 : 0.0));
  if (splits > 1) t += 3.0 + (double)(2 * splits * m * n * 4) / 4.0e6;
  return t;
}

constexpr int kMaxSplits = 16, kSplitStages = 8;  // ranges of a depth, least stages of one

inline Plan plan(const Cost& cost, int64_t m, int64_t n, int64_t stages) {
  Plan best{kSmall, 1, (int)stages};
  double least = plan_time(cost, m, n, stages, kSmall, 1);
  for (int tile = kBig; tile <= kSmall; ++tile)
    for (int64_t splits = 1; splits <= kMaxSplits; ++splits) {
      const int64_t per = ceil_div(stages, splits), used = ceil_div(stages, per);
      if (splits > 1 && per < kSplitStages) break;
      if (stages - (used - 1) * per < kMinStages[tile]) continue;  // the last range
      const double t = plan_time(cost, m, n, stages, tile, used);
      if (t < least) {
        least = t;
        best = {tile, (int)used, (int)per};
      }
    }
  return best;
}

// Raises a kernel's dynamic LDS limit once per process (one flag per kernel).
template <auto kern>
int allow_lds(size_t lds_bytes) {
  static std::once_flag once;
  static hipError_t rc = hipSuccess;
  std::call_once(once, [&] {
    rc = hipFuncSetAttribute(reinterpret_cast<const void*>(kern),
                             hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds_bytes);
  });
  DIONW_REQUIRE(rc == hipSuccess, "quantized product: hipFuncSetAttribute failed: %s", hipGetErrorString(rc));
  return kOk;
}

template <typename CFG, Form FORM, typename OUT>
int launch_tile(ProductArgs g, const Plan& p, hipStream_t stream) {
  constexpr auto kern = product_kernel<CFG, FORM, OUT>;
  DIONW_TRY(allow_lds<kern>(CFG::template lds_bytes<FORM>));
  const int64_t tm = ceil_div(g.m, CFG::BM), tn = ceil_div(g.n, CFG::BN);
  DIONW_REQUIRE(tm * tn < INT32_MAX / (8 * p.splits), "quantized product: too many tiles");
  g.tiles_m = (int32_t)tm;
  g.tiles_n = (int32_t)tn;
  g.xcd_group = CFG::BM == 256 && tm * tn >= 64 ? 32 : 0;
  g.per_split = p.per_split;
  const int total = (int)(tm * tn) * p.splits;
  size_t lds = CFG::template lds_bytes<FORM>;
  if constexpr (std::is_same<CFG, SmallTile>::value)
    lds = (size_t)std::min(CFG::ring, p.per_split) * CFG::template slot<FORM>;
  hipLaunchKernelGGL(kern, dim3((unsigned)round_up(total, 8)), dim3(CFG::threads), lds, stream, g, total);
  return check_launch("quantized product");
}

template <Form FORM, typename OUT>
int launch_tiles(const ProductArgs& g, const Plan& p, hipStream_t stream) {
  if (p.tile == kBig) return launch_tile<BigTile, FORM, OUT>(g, p, stream);
  if (p.tile == kMid) return launch_tile<MidTile, FORM, OUT>(g, p, stream);
  return launch_tile<SmallTile, FORM, OUT>(g, p, stream);
}

template <Form FORM, typename OUT>
int launch_product(const ProductArgs& g, const Plan& p, float* parts, hipStream_t stream) {
  const int64_t outputs = (int64_t)g.m * g.n;
  if (g.stages == 0) {
    DIONW_REQUIRE(ceil_div(outputs, 256) < INT32_MAX, "quantized product: too many outputs");
    hipLaunchKernelGGL(fill_bias_kernel<OUT>, dim3((unsigned)ceil_div(outputs, 256)), dim3(256), 0,
                       stream, g);
    return check_launch("fill_bias");
  }
  if (p.splits == 1) return launch_tiles<FORM, OUT>(g, p, stream);
  ProductArgs range = g;  // float32 sums of the depth's ranges, joined below
  range.c = parts;
  range.ldc = g.n;
  range.split_step = outputs;
  range.alpha = 1.f;
  range.bias = nullptr;
  DIONW_TRY((launch_tiles<FORM, float>(range, p, stream)));
  DIONW_REQUIRE(ceil_div(outputs, 1024) < INT32_MAX, "quantized product: too many outputs");
  hipLaunchKernelGGL(join_splits_kernel<OUT>, dim3((unsigned)ceil_div(outputs, 1024)), dim3(256), 0,
                     stream, g, parts, p.splits);
  return check_launch("join_splits");
}

}  // namespace
}  // namespace dionw

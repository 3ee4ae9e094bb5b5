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
// Both move 128 bytes of a row per stage, so that one tile serves them.
//
// Rows are dealt to fragments so that a lane's scales and outputs lie side by side: of the 16 F
// rows of a wave's F fragments, fragment f's lane i holds row F i + f. Then the F scale bytes
// of a lane are one LDS read, the instruction picks its byte (op_sel), and with the column
// operand first a lane ends with 8 consecutive columns of a row, which it stores at once.
#include "float8.h"

#include <algorithm>
#include <mutex>
#include <type_traits>

namespace dionw {
namespace {

typedef __attribute__((address_space(3))) void* lds_ptr_t;

struct ProductArgs {
  const uint8_t* a;        // rows of `stages` x 128 bytes at a pitch of lda bytes
  int64_t lda;
  const uint8_t* a_scale;  // codes: [stages][a_scale_ld] exponent bytes
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

// c += b a^T of a fragment pair; OA, OB: the scales' bytes.
template <bool CODES, int OA, int OB>
__device__ __forceinline__ void multiply(i32x8 b, i32x8 a, f32x4& c, int b_scale, int a_scale) {
  if constexpr (CODES) {
    c = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b, a, c, 0, 0, OB, b_scale, OA, a_scale);
  } else {
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
        __builtin_bit_cast(bf16x8, __builtin_shufflevector(b, b, 0, 1, 2, 3)),
        __builtin_bit_cast(bf16x8, __builtin_shufflevector(a, a, 0, 1, 2, 3)), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
        __builtin_bit_cast(bf16x8, __builtin_shufflevector(b, b, 4, 5, 6, 7)),
        __builtin_bit_cast(bf16x8, __builtin_shufflevector(a, a, 4, 5, 6, 7)), c, 0, 0, 0);
  }
}

// A fragment's two chunks of a lane.
__device__ __forceinline__ i32x8 chunks(const unsigned char* lo, const unsigned char* hi) {
  return __builtin_shufflevector(*reinterpret_cast<const i32x4*>(lo),
                                 *reinterpret_cast<const i32x4*>(hi), 0, 1, 2, 3, 4, 5, 6, 7);
}

// A stage's scale bytes of one operand's rows, straight to LDS: 4 a lane, 256 a load, those past
// the tile's `side` repeated. Even waves load the first operand's and odd ones the second's
// (several the same bytes), so that every wave issues one load. A block's bytes run to a
// multiple of 16, so a lane's 4 are in bounds; past the last it takes the last 4. All of them
// lie within 2^32 bytes (checked).
struct ScaleLoad {
#ifdef __HIP_DEVICE_COMPILE__
  __amdgpu_buffer_rsrc_t rsrc;
#endif
  uint32_t off, step;
  __device__ __forceinline__ ScaleLoad(const ProductArgs& g, int second, int row0, int side, int first,
                                       int n_stages, int lane) {
#ifdef __HIP_DEVICE_COMPILE__
    const uint8_t* at = second ? g.b_scale : g.a_scale;
    const int64_t ld = second ? g.b_scale_ld : g.a_scale_ld;
    step = (uint32_t)ld;
    off = (uint32_t)min((int64_t)row0 + min(4 * lane, side - 4), ld - 4);
    rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)(at + first * ld), 0, (uint32_t)(n_stages * ld), 0x00020000);
#endif
  }
  __device__ __forceinline__ void issue(int kt, unsigned char* to) const {
#ifdef __HIP_DEVICE_COMPILE__
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr_t)to, 4, off, (uint32_t)kt * step, 0, 0);
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
template <int F>
__device__ __forceinline__ int scale_bytes(uint32_t word, int i16) {
  return F == 4 ? (int)word : (int)(word >> (16 * (i16 & 1)));
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
// Bound: the board's power (8192^3 395 us, 2785 TFLOP/s, 366 sustained at 1387 W of 1400 and 1.8 GHz,
// the matrix pipe 77% busy; expanded 14336 x 4096 x 8192 720 us, 1336, at 1400 W and 2.05 GHz, 68%);
// at few stages the first loads and the stores (plan_time; 8192 x 2304 x 768 24 us, 20%).
template <int WM_, int WN_, int FI_, int FJ_>
struct QuadCfg {
  static constexpr int WM = WM_, WN = WN_, FI = FI_, FJ = FJ_;
  static constexpr int waves = WM * WN, threads = waves * 64;
  static constexpr int HM = WM * FI * 16, HN = WN * FJ * 16;  // half tile rows / columns
  static constexpr int BM = 2 * HM, BN = 2 * HN;
  static constexpr int half = HM * 128;        // bytes of a half stage
  static constexpr int L = half / 16 / threads;  // loads per lane
  static constexpr size_t lds_bytes = (size_t)8 * half + 2 * 512;
  static_assert(HM == HN && L >= 1 && FJ == 2, "square tiles, pairs of column fragments");
};

using BigTile = QuadCfg<2, 4, 4, 2>;  // 256x256
using MidTile = QuadCfg<2, 2, 2, 2>;  // 128x128

template <typename CFG, bool CODES, typename OUT>
__device__ __forceinline__ void quad_tile(const ProductArgs& g, int w) {
#ifdef __HIP_DEVICE_COMPILE__  // the host pass has no buffer-resource type
  constexpr int HM = CFG::HM, HN = CFG::HN, FI = CFG::FI, FJ = CFG::FJ, BM = CFG::BM, BN = CFG::BN;
  constexpr int L = CFG::L, W = CFG::waves, S = CODES ? 1 : 0;  // S: scale loads of a stage
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  unsigned char* lds_a = smem;                    // [buffer][half][HM][128]
  unsigned char* lds_b = smem + 4 * CFG::half;
  unsigned char* lds_s = smem + 8 * CFG::half;    // scales: [buffer][operand][256]

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
  const ScaleLoad scale_load(g, wave & 1, wave & 1 ? n0 : m0, BM, first, n_stages, lane);
  auto load_s = [&](int kt, int buf) {
    if constexpr (CODES) scale_load.issue(kt, lds_s + buf * 512 + (wave & 1) * 256);
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
    uint32_t a[2], b[2];  // by half: the words of scale_word
  };
  auto read_s = [&](Scales& s, int buf) {
    if constexpr (CODES) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        s.a[h] = scale_word<FI>(lds_s + buf * 512 + h * HM + wm * FI * 16, i16);
        s.b[h] = scale_word<FJ>(lds_s + buf * 512 + 256 + h * HN + wn * FJ * 16, i16);
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
  auto row = [&](auto qi_, auto qj_, auto i_, i32x8 (&b)[FJ], const int (&s)[2][2]) {
    constexpr int qi = decltype(qi_)::value, qj = decltype(qj_)::value, i = decltype(i_)::value;
    multiply<CODES, i, 0>(b[0], a[i], acc[qi * FI + i][qj * FJ], s[1][qj], s[0][qi]);
    multiply<CODES, i, 1>(b[1], a[i], acc[qi * FI + i][qj * FJ + 1], s[1][qj], s[0][qi]);
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
    int s[2][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      s[0][h] = scale_bytes<FI>(s0.a[h], i16);
      s[1][h] = scale_bytes<FJ>(s0.b[h], i16);
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
  static_assert((size_t)HM * HN * sizeof(OUT) <= CFG::lds_bytes, "a quadrant fits");
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
  static constexpr int slot = 2 * operand + 512;  // A, B, their scales
  static constexpr size_t lds_bytes = (size_t)ring * slot;
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

template <bool CODES, typename OUT>
__device__ __forceinline__ void small_tile(const ProductArgs& g, int w) {
#ifdef __HIP_DEVICE_COMPILE__
  using CFG = SmallTile;
  constexpr int R = CFG::ring, BM = CFG::BM, BN = CFG::BN, P = 4 + (CODES ? 1 : 0);
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
  const ScaleLoad scale_load(g, wave & 1, wave & 1 ? n0 : m0, BM, first, n_stages, lane);
  auto issue = [&](int kt) {
    unsigned char* stage = smem + (kt % R) * CFG::slot;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      __builtin_amdgcn_raw_ptr_buffer_load_lds(a_rsrc, (lds_ptr_t)(stage + (j * 4 + wave) * 1024), 16,
                                               a_off[j], kt * 128, 0, 0);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          b_rsrc, (lds_ptr_t)(stage + CFG::operand + (j * 4 + wave) * 1024), 16, b_off[j], kt * 128, 0, 0);
    }
    if constexpr (CODES) scale_load.issue(kt, stage + 2 * CFG::operand + (wave & 1) * 256);
  };
  const int G = lane >> 4, i16 = lane & 15, sw = (i16 >> 1) & 7;
  struct Frags {
    i32x8 a[2], b[2];
    uint32_t as, bs;
  };
  auto read = [&](Frags& f, int kt) {
    const unsigned char* stage = smem + (kt % R) * CFG::slot;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const unsigned char* at = stage + (i * 16 + i16) * 128;
      const unsigned char *ra = at + wm * 32 * 128, *rb = at + CFG::operand + wn * 32 * 128;
      f.a[i] = chunks(ra + ((G ^ sw) << 4), ra + (((4 + G) ^ sw) << 4));
      f.b[i] = chunks(rb + ((G ^ sw) << 4), rb + (((4 + G) ^ sw) << 4));
    }
    if constexpr (CODES) {
      const unsigned char* s = stage + 2 * CFG::operand;
      f.as = scale_word<2>(s + wm * 32, i16);
      f.bs = scale_word<2>(s + 256 + wn * 32, i16);
    } else {
      f.as = f.bs = 0;
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
    const int as = scale_bytes<2>(now.as, i16), bs = scale_bytes<2>(now.bs, i16);
    multiply<CODES, 0, 0>(now.b[0], now.a[0], acc[0][0], bs, as);
    multiply<CODES, 0, 1>(now.b[1], now.a[0], acc[0][1], bs, as);
    multiply<CODES, 1, 0>(now.b[0], now.a[1], acc[1][0], bs, as);
    multiply<CODES, 1, 1>(now.b[1], now.a[1], acc[1][1], bs, as);
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

template <typename CFG, bool CODES, typename OUT>
__global__ __launch_bounds__(CFG::threads, 1) __attribute__((amdgpu_waves_per_eu(2, 2))) void
float8_gemm_kernel(ProductArgs g, int total) {
  const int w = xcd_tile((int)blockIdx.x, total, g.xcd_group);
  if (w < 0) return;  // the whole workgroup: w depends on blockIdx only
  if constexpr (std::is_same<CFG, SmallTile>::value)
    small_tile<CODES, OUT>(g, w);
  else
    quad_tile<CFG, CODES, OUT>(g, w);
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
// depth is split, one more launch and the sums' way to memory and back. Measured, codes, us on 256 /
// 128 / 64 tiles: 8192^3 395 / 448 / 1338, 8192 x 14336 x 4096 358 / 423 / 1285, 4096^3 56 / 63 / 186;
// 8192 x 2304 x 768 28 / 23 / 71, 3001 x 1408 x 2048 25 / 16 / 35, 2048^3 24 / 11 / 29; 64 x 14336 x
// 4096 39 / 19 / 14, 1024^3 15 / 7.0 / 6.1, 512^3 11 / 5.7 / 4.7. Split in 1 / 2 / 4 / 8, 128 tiles:
// 100 x 4096 x 14336 48 / 32 / 23 / 22, expanded 2304 x 768 x 8192 56 / 41 / 41 / 48. The rule takes the
// fastest on all of them.
double plan_time(int64_t m, int64_t n, int64_t stages, int tile, int64_t splits) {
  constexpr double stage[3] = {1.4, 0.42, 0.28}, fixed[3] = {5.0, 1.0, 0.6};
  const int64_t per = ceil_div(stages, splits);
  const int64_t rounds = ceil_div(ceil_div(m, kSide[tile]) * ceil_div(n, kSide[tile]) * splits, 256);
  double t = (double)rounds * (stage[tile] * (double)per + fixed[tile] +
                               (tile == kSmall && rounds > 1 ? 1.4 : 0.0));
  if (splits > 1) t += 3.0 + (double)(2 * splits * m * n * 4) / 4.0e6;
  return t;
}

constexpr int kMaxSplits = 16, kSplitStages = 8;  // ranges of a depth, least stages of one

Plan plan(int64_t m, int64_t n, int64_t stages) {
  Plan best{kSmall, 1, (int)stages};
  double least = plan_time(m, n, stages, kSmall, 1);
  for (int tile = kBig; tile <= kSmall; ++tile)
    for (int64_t splits = 1; splits <= kMaxSplits; ++splits) {
      const int64_t per = ceil_div(stages, splits), used = ceil_div(stages, per);
      if (splits > 1 && per < kSplitStages) break;
      if (stages - (used - 1) * per < kMinStages[tile]) continue;  // the last range
      const double t = plan_time(m, n, stages, tile, used);
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
  DIONW_REQUIRE(rc == hipSuccess, "float8_gemm: hipFuncSetAttribute failed: %s", hipGetErrorString(rc));
  return kOk;
}

template <typename CFG, bool CODES, typename OUT>
int launch_tile(ProductArgs g, const Plan& p, hipStream_t stream) {
  constexpr auto kern = float8_gemm_kernel<CFG, CODES, OUT>;
  DIONW_TRY(allow_lds<kern>(CFG::lds_bytes));
  const int64_t tm = ceil_div(g.m, CFG::BM), tn = ceil_div(g.n, CFG::BN);
  DIONW_REQUIRE(tm * tn < INT32_MAX / (8 * p.splits), "float8_gemm: too many tiles");
  g.tiles_m = (int32_t)tm;
  g.tiles_n = (int32_t)tn;
  g.xcd_group = CFG::BM == 256 && tm * tn >= 64 ? 32 : 0;
  g.per_split = p.per_split;
  const int total = (int)(tm * tn) * p.splits;
  size_t lds = CFG::lds_bytes;
  if constexpr (std::is_same<CFG, SmallTile>::value)
    lds = (size_t)std::min(CFG::ring, p.per_split) * CFG::slot;
  hipLaunchKernelGGL(kern, dim3((unsigned)round_up(total, 8)), dim3(CFG::threads), lds, stream, g, total);
  return check_launch("float8_gemm");
}

template <bool CODES, typename OUT>
int launch_tiles(const ProductArgs& g, const Plan& p, hipStream_t stream) {
  if (p.tile == kBig) return launch_tile<BigTile, CODES, OUT>(g, p, stream);
  if (p.tile == kMid) return launch_tile<MidTile, CODES, OUT>(g, p, stream);
  return launch_tile<SmallTile, CODES, OUT>(g, p, stream);
}

template <bool CODES, typename OUT>
int launch_product(const ProductArgs& g, const Plan& p, float* parts, hipStream_t stream) {
  const int64_t outputs = (int64_t)g.m * g.n;
  if (g.stages == 0) {
    DIONW_REQUIRE(ceil_div(outputs, 256) < INT32_MAX, "float8_gemm: too many outputs");
    hipLaunchKernelGGL(fill_bias_kernel<OUT>, dim3((unsigned)ceil_div(outputs, 256)), dim3(256), 0,
                       stream, g);
    return check_launch("float8_fill_bias");
  }
  if (p.splits == 1) return launch_tiles<CODES, OUT>(g, p, stream);
  ProductArgs range = g;  // float32 sums of the depth's ranges, joined below
  range.c = parts;
  range.ldc = g.n;
  range.split_step = outputs;
  range.alpha = 1.f;
  range.bias = nullptr;
  DIONW_TRY((launch_tiles<CODES, float>(range, p, stream)));
  DIONW_REQUIRE(ceil_div(outputs, 1024) < INT32_MAX, "float8_gemm: too many outputs");
  hipLaunchKernelGGL(join_splits_kernel<OUT>, dim3((unsigned)ceil_div(outputs, 1024)), dim3(256), 0,
                     stream, g, parts, p.splits);
  return check_launch("float8_join_splits");
}

}  // namespace
}  // namespace dionw

using namespace dionw;

extern "C" {

int dionw_float8_gemm_plan(int32_t expanded, int64_t m, int64_t n, int64_t depth, int32_t* side,
                           int32_t* ranges) {
  DIONW_REQUIRE(m > 0 && n > 0 && depth > 0 && depth % kTile == 0 && side && ranges,
                "float8_gemm_plan: bad arguments");
  const Plan p = plan(m, n, depth / kTile * (expanded ? 2 : 1));
  *side = kSide[p.tile];
  *ranges = p.splits;
  return kOk;
}

size_t dionw_float8_gemm_workspace(int32_t expanded, int64_t m, int64_t n, int64_t depth) {
  if (m <= 0 || n <= 0 || depth <= 0 || depth % kTile) return 0;
  const Plan p = plan(m, n, depth / kTile * (expanded ? 2 : 1));
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
  const Plan p = depth ? plan(m, n, row / 128) : Plan{kSmall, 1, 1};
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
  if (elem == kF16) return launch_product<true, _Float16>(g, p, parts, stream);
  if (elem == kBF16) return launch_product<true, __bf16>(g, p, parts, stream);
  return launch_product<false, float>(g, p, parts, stream);
}

}  // extern "C"

// Multi-tensor AdamW whose moments are held in 8 bits.
//
// Per element, with m the first moment and r the root of the second:
//
//   m = b1 m0 + (1 - b1) g        r = sqrt(b2 r0^2 + (1 - b2) g^2)
//   p = p (1 - lr wd) - step_size m / (r root + eps)
//   step_size = lr / (1 - b1^t)   root = 1 / sqrt(1 - b2^t)
//
// all in float32, every operation rounded on its own (contraction off) but for p's one
// fused multiply-add, so that the codes do not depend on how a compiler fuses the formula.
//
// Formats. m is e4m3 (sign, 4 exponent bits, bias 7, 3 fraction bits; largest 448,
// subnormal unit 2^-9); r is an unsigned float of 4 exponent bits (bias 8) and 4 fraction
// bits (largest 248, unit 2^-11): the root of v needs half of v's range and no sign, so it
// keeps one bit more than e4m3 would. 256 consecutive elements share a scale of each: the
// smallest power of two that brings their largest magnitude to the format's largest value
// at most. A power of two costs no fraction bit in a floating format, scales without
// rounding, and an element that did not change keeps its code whatever its neighbours do.
//
// Rounding is stochastic: up where the dropped part, in units of the last place, is at
// least 1 - R / 2^16. R comes from a hash of (step, tensor, element), so a run repeats bit
// for bit and no generator state has to be kept. To nearest, an average that moves by less
// than half a code per step stands still (b2 = 0.999 moves r by 0.05%, half a code is 1.6
// to 3.1%); stochastically it moves as it should in the mean. A code of r is never rounded
// to zero from above: r is the divisor.
//
// An element whose new m or second moment is not finite is stored as NaN in m (its
// parameter is NaN at this step or the next) and takes no part in its block's scales.
//
// Bound: HBM, 16 B an element (p read and written, g read, two codes read and written)
// against 28 with float32 moments. A wave loads 4 blocks of 256 before its first store, the
// division of work that streams the float32 pass best. 525 M elements: 1464 us (5.74 TB/s; the
// float32 pass 2580), 38.6 M: 112 us; the moments' values (2 B read, 8 written) 965 and 66 us.
#include "common.h"

#include <cmath>

namespace dionw {
namespace {

#pragma clang fp contract(off)

constexpr int kBlock = 256;       // elements that share a scale: a wave, 4 a lane
constexpr int kBlocks = 4;        // blocks of a wave, all loads before the first store
constexpr int kChunk = 4 * kBlocks * kBlock;  // elements of a workgroup of 4 waves
constexpr int kMaxTable = 80;     // tensors of a launch (3.6 KB of kernel arguments)

struct Table {
  float* p[kMaxTable];
  const float* g[kMaxTable];
  float* shadow[kMaxTable];      // EMA shadows (fused EMA)
  int64_t numel[kMaxTable];
  int64_t block0[kMaxTable];     // first state block of the tensor
  int32_t chunk0[kMaxTable + 1]; // first chunk
  int32_t id[kMaxTable];         // place of the tensor's step
  int count;
};

struct State {
  uint32_t* m;       // four codes a word
  float* m_scale;
  uint32_t* r;
  float* r_scale;
  const float* scalars;  // [tensor][4]: step_size, root, hash key (bits), unused
};

struct Scalars {
  float beta1, one_beta1, beta2, one_beta2, eps, decay;
};

__device__ __forceinline__ int find_tensor(const int32_t* chunk0, int count, int chunk) {
  int lo = 0, hi = count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (chunk0[mid] <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// 32 bits from 32: two rounds of multiply and xor-shift.
__device__ __forceinline__ uint32_t mix(uint32_t x) {
  x ^= x >> 16;
  x *= 0x9E3779B1u;
  x ^= x >> 15;
  x *= 0x85EBCA77u;
  return x ^ (x >> 16);
}

__device__ __forceinline__ float power(uint32_t byte) { return __uint_as_float(byte << 23); }

// The exponent byte of the scale of a block whose largest magnitude has the bits `largest`:
// `carry` takes a fraction above the format's largest into the next binade, `top` is the
// largest value's binade. At least 1, so that the scale and its reciprocal are normal.
__device__ __forceinline__ uint32_t scale_byte(uint32_t largest, uint32_t carry, uint32_t top) {
  const uint32_t field = (largest + carry) >> 23;
  return field > top ? field - top : 1u;
}
__device__ __forceinline__ uint32_t m_byte(uint32_t largest) { return scale_byte(largest, 0x1FFFFFu, 8); }
__device__ __forceinline__ uint32_t r_byte(uint32_t largest) { return scale_byte(largest, 0x07FFFFu, 7); }

// The code of a magnitude u in units of its scale, rounded up by noise / 2^16: FRACTION
// fraction bits, exponent bias BIAS. Normal values take the float32 fields (the noise sits
// right below the last kept bit, a carry runs into the exponent); subnormal ones are whole
// units of 2^(1 - BIAS - FRACTION).
template <int FRACTION, int BIAS>
__device__ __forceinline__ uint32_t encode(float u, uint32_t noise) {
  const uint32_t normal =
      (__float_as_uint(u) - ((127u - BIAS) << 23) + (noise << (7 - FRACTION))) >> (23 - FRACTION);
  constexpr float kUnits = (float)(1 << (16 + BIAS - 1 + FRACTION));
  constexpr float kNormal = 2.f / (float)(1 << BIAS);
  const uint32_t small = ((uint32_t)(fminf(u, kNormal) * kUnits) + noise) >> 16;
  return u < kNormal ? small : normal;
}

__device__ __forceinline__ float r_value(uint32_t code) {
  const float normal = __uint_as_float((code << 19) + (119u << 23));
  return code < 16u ? (float)code * 0x1p-11f : normal;
}

template <int BYTE>
__device__ __forceinline__ float m_value(uint32_t codes) {
  return __builtin_amdgcn_cvt_f32_fp8((int)codes, BYTE);
}
__device__ __forceinline__ void m_values(uint32_t codes, float (&v)[4]) {
  v[0] = m_value<0>(codes);
  v[1] = m_value<1>(codes);
  v[2] = m_value<2>(codes);
  v[3] = m_value<3>(codes);
}

__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, off, kWave));
  return v;
}

// steps[id] += 1 and what the element pass needs of it.
struct Ids {
  int32_t id[256];
  int count;
};
__global__ void adamw_8bit_scalars_kernel(Ids ids, float* steps, float* scalars, double lr,
                                          double beta1, double beta2) {
  const int i = threadIdx.x;
  if (i >= ids.count) return;
  const int id = ids.id[i];
  const float t = steps[id] + 1.f;
  steps[id] = t;
  scalars[4 * id] = (float)(lr / (1 - ::pow(beta1, (double)t)));
  scalars[4 * id + 1] = (float)(1 / std::sqrt(1 - ::pow(beta2, (double)t)));
  scalars[4 * id + 2] = __uint_as_float(mix((uint32_t)id * 0x9E3779B1u + (uint32_t)t));
}

template <bool EMA>
__global__ __launch_bounds__(256) void adamw_8bit_kernel(Table t, State state, Scalars s,
                                                         float ema_weight) {
  const int tensor = find_tensor(t.chunk0, t.count, blockIdx.x);
  const int64_t first = (int64_t)(blockIdx.x - t.chunk0[tensor]) * kChunk;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t numel = t.numel[tensor];
  const int id = t.id[tensor];
  float* p = t.p[tensor];
  const float* g = t.g[tensor];
  float* sh = EMA ? t.shadow[tensor] : nullptr;
  const bool vec = ((reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(g) |
                     reinterpret_cast<uintptr_t>(sh)) & 15) == 0;

  f32x4 pv[kBlocks], gv[kBlocks], sv[kBlocks];
  uint32_t mc[kBlocks], rc[kBlocks];
  float ms[kBlocks], rs[kBlocks];
#pragma unroll
  for (int b = 0; b < kBlocks; ++b) {
    const int64_t at = first + (b * 4 + wave) * kBlock;  // the wave's block in the tensor
    if (at >= numel) break;
    const int64_t block = t.block0[tensor] + at / kBlock;
    const int64_t e = at + 4 * lane;
    mc[b] = __builtin_nontemporal_load(state.m + block * 64 + lane);
    rc[b] = __builtin_nontemporal_load(state.r + block * 64 + lane);
    ms[b] = state.m_scale[block];
    rs[b] = state.r_scale[block];
    if (vec && e + 4 <= numel) {
      pv[b] = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(p + e));
      gv[b] = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(g + e));
      if (EMA) sv[b] = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(sh + e));
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const bool in = e + k < numel;
        pv[b][k] = in ? p[e + k] : 0.f;
        gv[b][k] = in ? g[e + k] : 0.f;
        if (EMA) sv[b][k] = in ? sh[e + k] : 0.f;
      }
    }
  }
  const float step_size = state.scalars[4 * id], root = state.scalars[4 * id + 1];
  const uint32_t key0 = __float_as_uint(state.scalars[4 * id + 2]);
#pragma unroll
  for (int b = 0; b < kBlocks; ++b) {
    const int64_t at = first + (b * 4 + wave) * kBlock;
    if (at >= numel) break;
    const int64_t block = t.block0[tensor] + at / kBlock;
    const int64_t e = at + 4 * lane;
    float m[4], r[4];
    m_values(mc[b], m);
    uint32_t m_most = 0, r_most = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float gk = gv[b][k];
      const float r0 = r_value((rc[b] >> (8 * k)) & 255u) * rs[b];
      m[k] = m[k] * ms[b] * s.beta1 + gk * s.one_beta1;
      r[k] = std::sqrt(r0 * r0 * s.beta2 + gk * s.one_beta2 * gk);
      pv[b][k] = __builtin_fmaf(pv[b][k], s.decay, -(m[k] * step_size / (r[k] * root + s.eps)));
      const uint32_t mb = __float_as_uint(m[k]) & 0x7FFFFFFFu, rb = __float_as_uint(r[k]);
      if (mb < 0x7F800000u && rb < 0x7F800000u) {
        m_most = max(m_most, mb);
        r_most = max(r_most, rb);
      }
    }
    const uint32_t mby = m_byte(wave_max(m_most)), rby = r_byte(wave_max(r_most));
    const float m_inv = power(254 - mby), r_inv = power(254 - rby);
    const uint32_t key = mix(key0 + (uint32_t)(e >> 32));
    uint32_t mw = 0, rw = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t noise = mix((uint32_t)(e + k) ^ key);
      const uint32_t mb = __float_as_uint(m[k]), rb = __float_as_uint(r[k]);
      const bool finite = (mb & 0x7FFFFFFFu) < 0x7F800000u && rb < 0x7F800000u;
      uint32_t mk = encode<3, 7>(fabsf(m[k]) * m_inv, noise & 0xFFFFu) | ((mb >> 24) & 0x80u);
      uint32_t rk = encode<4, 8>(r[k] * r_inv, noise >> 16);
      if (rk == 0 && rb != 0) rk = 1;
      mw |= (finite ? mk : 0x7Fu) << (8 * k);
      rw |= (finite ? rk : 0xFFu) << (8 * k);
    }
    __builtin_nontemporal_store(mw, state.m + block * 64 + lane);
    __builtin_nontemporal_store(rw, state.r + block * 64 + lane);
    if (lane == 0) {
      state.m_scale[block] = power(mby);
      state.r_scale[block] = power(rby);
    }
    if (EMA) {
#pragma unroll
      for (int k = 0; k < 4; ++k) sv[b][k] = ema_lerp(sv[b][k], pv[b][k], ema_weight);
    }
    if (vec && e + 4 <= numel) {
      __builtin_nontemporal_store(pv[b], reinterpret_cast<f32x4*>(p + e));
      if (EMA) __builtin_nontemporal_store(sv[b], reinterpret_cast<f32x4*>(sh + e));
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (e + k < numel) {
          p[e + k] = pv[b][k];
          if (EMA) sh[e + k] = sv[b][k];
        }
    }
  }
}

// The values the codes stand for, tensor after tensor.
struct ValuesTable {
  int64_t numel[kMaxTable];
  int64_t block0[kMaxTable];
  int64_t out0[kMaxTable];
  int32_t chunk0[kMaxTable + 1];
  int count;
};

__global__ __launch_bounds__(256) void adamw_8bit_values_kernel(ValuesTable t, State state,
                                                                float* exp_avg, float* rms) {
  const int tensor = find_tensor(t.chunk0, t.count, blockIdx.x);
  const int64_t first = (int64_t)(blockIdx.x - t.chunk0[tensor]) * kChunk;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t numel = t.numel[tensor];
  float* mo = exp_avg + t.out0[tensor];
  float* ro = rms + t.out0[tensor];
  const bool vec = ((reinterpret_cast<uintptr_t>(mo) | reinterpret_cast<uintptr_t>(ro)) & 15) == 0;
  uint32_t mc[kBlocks], rc[kBlocks];
  float ms[kBlocks], rs[kBlocks];
#pragma unroll
  for (int b = 0; b < kBlocks; ++b) {
    const int64_t at = first + (b * 4 + wave) * kBlock;
    if (at >= numel) break;
    const int64_t block = t.block0[tensor] + at / kBlock;
    mc[b] = state.m[block * 64 + lane];
    rc[b] = state.r[block * 64 + lane];
    ms[b] = state.m_scale[block];
    rs[b] = state.r_scale[block];
  }
#pragma unroll
  for (int b = 0; b < kBlocks; ++b) {
    const int64_t at = first + (b * 4 + wave) * kBlock;
    if (at >= numel) break;
    const int64_t e = at + 4 * lane;
    float m[4];
    m_values(mc[b], m);
    f32x4 mv, rv;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      mv[k] = m[k] * ms[b];
      rv[k] = r_value((rc[b] >> (8 * k)) & 255u) * rs[b];
    }
    if (vec && e + 4 <= numel) {
      __builtin_nontemporal_store(mv, reinterpret_cast<f32x4*>(mo + e));
      __builtin_nontemporal_store(rv, reinterpret_cast<f32x4*>(ro + e));
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (e + k < numel) {
          mo[e + k] = mv[k];
          ro[e + k] = rv[k];
        }
    }
  }
}

// Appends tensor i to a launch; false where the launch is full.
template <typename TABLE>
bool append(TABLE& t, int32_t& chunks, int64_t numel, int64_t block0) {
  const int64_t c = ceil_div(numel, kChunk);
  if (t.count == kMaxTable || chunks + c > INT32_MAX / 2) return false;
  t.numel[t.count] = numel;
  t.block0[t.count] = block0;
  t.chunk0[t.count] = chunks;
  chunks += (int32_t)c;
  ++t.count;
  t.chunk0[t.count] = chunks;
  return true;
}

int check_tensor(const char* what, int i, int64_t numel, int64_t block0, int64_t blocks) {
  DIONW_REQUIRE(numel >= 0 && ceil_div(numel, kChunk) <= INT32_MAX / 2, "%s: bad size of tensor %d",
                what, i);
  DIONW_REQUIRE(block0 >= 0 && block0 <= blocks && ceil_div(numel, kBlock) <= blocks - block0,
                "%s: the state blocks of tensor %d lie outside the state", what, i);
  return kOk;
}

int check_state(const char* what, const void* m, const void* ms, const void* r, const void* rs) {
  DIONW_REQUIRE(m && ms && r && rs, "%s: null state", what);
  DIONW_REQUIRE(((reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(r) |
                  reinterpret_cast<uintptr_t>(ms) | reinterpret_cast<uintptr_t>(rs)) & 3) == 0,
                "%s: the state must be 4-byte aligned", what);
  return kOk;
}

}  // namespace
}  // namespace dionw

using namespace dionw;

extern "C" {

int dionw_adamw_8bit(float* const* params, const float* const* grads, float* const* shadows,
                     const int64_t* numels, const int64_t* first_blocks, const int32_t* ids,
                     int32_t count, int64_t blocks, int32_t tensors, void* exp_avg,
                     float* exp_avg_scale, void* rms, float* rms_scale, float* steps,
                     float* scalars, double lr, double beta1, double beta2, double weight_decay,
                     double eps, float ema_weight, hipStream_t stream) {
  DIONW_REQUIRE(count >= 0 && blocks >= 0 && tensors >= 0, "adamw_8bit: negative count");
  if (count == 0) return kOk;
  DIONW_REQUIRE(params && grads && numels && first_blocks && ids && steps && scalars,
                "adamw_8bit: null table");
  DIONW_TRY(check_state("adamw_8bit", exp_avg, exp_avg_scale, rms, rms_scale));
  for (int32_t i = 0; i < count; ++i) {
    DIONW_REQUIRE(numels[i] == 0 || (params[i] && grads[i] && (!shadows || shadows[i])),
                  "adamw_8bit: null pointer in tensor %d", i);
    DIONW_REQUIRE(ids[i] >= 0 && ids[i] < tensors, "adamw_8bit: bad id of tensor %d", i);
    DIONW_TRY(check_tensor("adamw_8bit", i, numels[i], first_blocks[i], blocks));
  }
  for (int32_t start = 0; start < count; start += 256) {
    Ids table{};
    table.count = count - start < 256 ? count - start : 256;
    for (int i = 0; i < table.count; ++i) table.id[i] = ids[start + i];
    hipLaunchKernelGGL(adamw_8bit_scalars_kernel, dim3(1), dim3(256), 0, stream, table, steps,
                       scalars, lr, beta1, beta2);
    DIONW_TRY(check_launch("adamw_8bit_scalars"));
  }
  const State state{static_cast<uint32_t*>(exp_avg), exp_avg_scale, static_cast<uint32_t*>(rms),
                    rms_scale, scalars};
  const Scalars s{(float)beta1, (float)(1 - beta1), (float)beta2, (float)(1 - beta2), (float)eps,
                  (float)(1 - lr * weight_decay)};
  for (int32_t i = 0; i < count;) {
    Table t{};
    int32_t chunks = 0;
    for (; i < count; ++i) {
      if (numels[i] == 0) continue;
      if (!append(t, chunks, numels[i], first_blocks[i])) break;
      t.p[t.count - 1] = params[i];
      t.g[t.count - 1] = grads[i];
      t.shadow[t.count - 1] = shadows ? shadows[i] : nullptr;
      t.id[t.count - 1] = ids[i];
    }
    if (t.count == 0) continue;
    if (shadows)
      hipLaunchKernelGGL(adamw_8bit_kernel<true>, dim3((unsigned)chunks), dim3(256), 0, stream, t,
                         state, s, ema_weight);
    else
      hipLaunchKernelGGL(adamw_8bit_kernel<false>, dim3((unsigned)chunks), dim3(256), 0, stream, t,
                         state, s, 0.f);
    DIONW_TRY(check_launch("adamw_8bit"));
  }
  return kOk;
}

int dionw_adamw_8bit_values(const int64_t* numels, const int64_t* first_blocks, int32_t count,
                            int64_t blocks, const void* exp_avg, const float* exp_avg_scale,
                            const void* rms, const float* rms_scale, float* exp_avg_out,
                            float* rms_out, hipStream_t stream) {
  DIONW_REQUIRE(count >= 0 && blocks >= 0, "adamw_8bit_values: negative count");
  if (count == 0) return kOk;
  DIONW_REQUIRE(numels && first_blocks && exp_avg_out && rms_out, "adamw_8bit_values: null table");
  DIONW_TRY(check_state("adamw_8bit_values", exp_avg, exp_avg_scale, rms, rms_scale));
  for (int32_t i = 0; i < count; ++i)
    DIONW_TRY(check_tensor("adamw_8bit_values", i, numels[i], first_blocks[i], blocks));
  const State state{static_cast<uint32_t*>(const_cast<void*>(exp_avg)),
                    const_cast<float*>(exp_avg_scale),
                    static_cast<uint32_t*>(const_cast<void*>(rms)), const_cast<float*>(rms_scale),
                    nullptr};
  int64_t out = 0;
  for (int32_t i = 0; i < count;) {
    ValuesTable t{};
    int32_t chunks = 0;
    for (; i < count; ++i) {
      if (numels[i] == 0) continue;
      if (!append(t, chunks, numels[i], first_blocks[i])) break;
      t.out0[t.count - 1] = out;
      out += numels[i];
    }
    if (t.count == 0) continue;
    hipLaunchKernelGGL(adamw_8bit_values_kernel, dim3((unsigned)chunks), dim3(256), 0, stream, t,
                       state, exp_avg_out, rms_out);
    DIONW_TRY(check_launch("adamw_8bit_values"));
  }
  return kOk;
}

}  // extern "C"

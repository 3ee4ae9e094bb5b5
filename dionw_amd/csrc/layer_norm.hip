// Layer norm of rows, its gradients, and the norm whose output is quantized to 4 bits as it is made.
//
//   u = (x - mean(x)) / sqrt(var(x) + eps)        y = u g + b
//   dx = (w - mean(w) - u mean(w u)) / sqrt(var(x) + eps), w = dy g
//   dg = sum of dy u over the rows                db = sum of dy over the rows
//
// Rows are held in registers from their one reading on, so that the variance is that of the values
// minus their mean, not a difference of sums: rows far from zero keep their digits. Statistics and
// sums are float32, in a fixed order.
#include "float4.h"

#include <algorithm>

namespace dionw {
namespace {

// Threads of a workgroup whose rows take LANES threads each: one row, or 256 threads of rows of a wave.
constexpr int threads_of(int lanes) { return lanes > kWave ? lanes : 256; }

struct NormArgs {
  const void* x;
  int64_t x_ld, rows, cols;
  const void *weight, *bias;  // null: ones, zeros
  int32_t w_elem, b_elem;
  float eps;
  void* y;                 // [rows][cols]
  float *mean, *rstd;      // [rows] each, or null
  uint8_t *data, *scale;   // 4-bit output instead of y
  int64_t depth, scale_ld;
};

// ---- 8 columns of a row ------------------------------------------------------------------

// 8 parameters as float32; `left` of them are there.
template <typename T>
__device__ __forceinline__ void values8(const void* at, int64_t c, int64_t left, float (&v)[8]) {
  Square<T> s;
  const T* p = reinterpret_cast<const T*>(at) + c;
  if (left >= 8) s.load(0, p);
  else s.load(0, p, left);
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = s.value(0, k);
}
__device__ __forceinline__ void parameters8(const void* at, int32_t elem, int64_t c, int64_t left,
                                            float fill, float (&v)[8]) {
  if (!at) {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = fill;
  } else if (elem == kF32) {
    values8<float>(at, c, left, v);
  } else if (elem == kBF16) {
    values8<__bf16>(at, c, left, v);
  } else {
    values8<_Float16>(at, c, left, v);
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* at, const float (&v)[8], int64_t left) {
  if (left >= 8) {
    constexpr int N = 16 / sizeof(T);
    typedef T line __attribute__((ext_vector_type(N)));
    typedef T anywhere __attribute__((ext_vector_type(N), aligned(sizeof(T))));
#pragma unroll
    for (int h = 0; h < 8 / N; ++h) {
      line o;
#pragma unroll
      for (int k = 0; k < N; ++k) o[k] = (T)v[h * N + k];
      *reinterpret_cast<anywhere*>(at + h * N) = o;
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < left) at[k] = (T)v[k];
  }
}

// The sum over a row's LANES threads, in each of them; `sums`: LDS of its own for more than a wave.
template <int LANES>
__device__ __forceinline__ float row_sum(float v, float* sums) {
#pragma unroll
  for (int off = (LANES < kWave ? LANES : kWave) / 2; off >= 1; off >>= 1) v += __shfl_xor(v, off, kWave);
  if constexpr (LANES > kWave) {
    constexpr int W = LANES / kWave;
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) v += sums[w];
  }
  return v;
}

// ---- forward ------------------------------------------------------------------------------
//
// LANES threads a row, K chunks of 8 columns a thread, `LANES * 8 * K` columns at most.
// Bound: HBM, x read and y written: 8192 x 4096 bfloat16 24 us (5.6 TB/s); float32 41 again and again, its x then
// from the Infinity Cache, 59 (4.5) in a training pass. To 4 bits not HBM: 26 us for 85 MB (3.3 TB/s; quantizing such
// rows alone takes 13.8). A workgroup takes one row, meets twice with no other row of its own on its way, and reads
// 32 KB of parameters beside 8 KB of x. 8192 x 768 float32 10, 2048 x 16384 bfloat16 32.

// Workgroup b's first row. 4-bit output: the rows whose scales share a line of memory run on one XCD
// (the hardware deals workgroup b to XCD b % 8), whose L2 then writes the line once.
template <bool CODES>
__device__ __forceinline__ int64_t first_row(uint32_t b, int rows_each, uint32_t groups) {
  if (!CODES) return (int64_t)b * rows_each;
  const uint32_t run = 64 / rows_each, turn = 8 * run, whole = groups / turn * turn;
  if (b >= whole) return (int64_t)b * rows_each;
  const uint32_t x = b % 8, i = b % turn / 8;
  return (int64_t)(b / turn * turn + x * run + i) * rows_each;
}

template <typename T, bool CODES>
__device__ __forceinline__ void write8(const NormArgs& g, int64_t row, int64_t c, float (&v)[8]) {
  if constexpr (CODES) {
    uint32_t most = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (c + k >= g.cols) v[k] = 0.f;
      most = max(most, __float_as_uint(v[k]) & 0x7FFFFFFFu);
    }
    const uint32_t byte = scale_byte4<false>(largest_of_four(most));
    const float scale = power(byte);
    uint32_t w = codes2<0>(0, v[0], v[1], scale);
    w = codes2<1>(w, v[2], v[3], scale);
    w = codes2<2>(w, v[4], v[5], scale);
    w = codes2<3>(w, v[6], v[7], scale);
    if (row < g.rows && c < g.depth) {
      *reinterpret_cast<uint32_t*>(g.data + row * (g.depth / 2) + c / 2) = w;
      if (c % kBlock4 == 0) g.scale[c / kBlock4 * g.scale_ld + row] = (uint8_t)byte;
    }
  } else {
    if (row < g.rows) store8<T>(reinterpret_cast<T*>(g.y) + row * g.cols + c, v, g.cols - c);
  }
}

template <typename T, int LANES, int K, bool CODES>
__global__ __launch_bounds__(threads_of(LANES)) void norm_kernel(NormArgs g) {
  constexpr int kEach = threads_of(LANES) / LANES;
  __shared__ float sums[2][LANES / kWave + 1];
  const int lane = threadIdx.x % LANES;
  const int64_t row = first_row<CODES>(blockIdx.x, kEach, gridDim.x) + threadIdx.x / LANES;
  Square<T> v;  // K of its rows
  const T* at = reinterpret_cast<const T*>(g.x) + min(row, g.rows - 1) * g.x_ld;
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int64_t c = 8 * (lane + k * LANES);
    if (c + 8 <= g.cols) v.load(k, at + c);
    else v.load(k, at + c, g.cols - c);
  }
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int e = 0; e < 8; ++e) s += v.value(k, e);
  const float mean = row_sum<LANES>(s, sums[0]) / (float)g.cols;
  s = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int64_t c = 8 * (lane + k * LANES);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float d = c + e < g.cols ? v.value(k, e) - mean : 0.f;
      s = __builtin_fmaf(d, d, s);
    }
  }
  const float rstd = 1.f / sqrtf(row_sum<LANES>(s, sums[1]) / (float)g.cols + g.eps);
  if (!CODES && g.mean && lane == 0 && row < g.rows) {
    g.mean[row] = mean;
    g.rstd[row] = rstd;
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int64_t c = 8 * (lane + k * LANES);
    if (!CODES && c >= g.cols) continue;
    float gain[8], bias[8], y[8];
    parameters8(g.weight, g.w_elem, c, g.cols - c, 1.f, gain);
    parameters8(g.bias, g.b_elem, c, g.cols - c, 0.f, bias);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = __builtin_fmaf((v.value(k, e) - mean) * rstd, gain[e], bias[e]);
    write8<T, CODES>(g, row, c, y);
  }
}

// Rows past the registers of a workgroup are read three times.
constexpr int kWide = 1024;
template <typename T, bool CODES>
__global__ __launch_bounds__(kWide) void norm_wide_kernel(NormArgs g) {
  __shared__ float sums[2][kWide / kWave];
  const int64_t row = first_row<CODES>(blockIdx.x, 1, gridDim.x), end = CODES ? g.depth : g.cols;
  const T* at = reinterpret_cast<const T*>(g.x) + row * g.x_ld;
  auto sweep = [&](auto body, int64_t last) {
    for (int64_t c = 8 * threadIdx.x; c < last; c += 8 * kWide) {
      float v[8];
      values8<T>(at, c, g.cols - c, v);
      body(c, v);
    }
  };
  float s = 0.f;
  sweep([&](int64_t, float (&v)[8]) {
    s += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
  }, g.cols);
  const float mean = row_sum<kWide>(s, sums[0]) / (float)g.cols;
  s = 0.f;
  sweep([&](int64_t c, float (&v)[8]) {
    float part = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float d = c + e < g.cols ? v[e] - mean : 0.f;
      part = __builtin_fmaf(d, d, part);
    }
    s += part;
  }, g.cols);
  const float rstd = 1.f / sqrtf(row_sum<kWide>(s, sums[1]) / (float)g.cols + g.eps);
  if (!CODES && g.mean && threadIdx.x == 0) {
    g.mean[row] = mean;
    g.rstd[row] = rstd;
  }
  sweep([&](int64_t c, float (&v)[8]) {  // a block's 4 lanes together: depth is a multiple of 256
    float gain[8], bias[8], y[8];
    parameters8(g.weight, g.w_elem, c, g.cols - c, 1.f, gain);
    parameters8(g.bias, g.b_elem, c, g.cols - c, 0.f, bias);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = __builtin_fmaf((v[e] - mean) * rstd, gain[e], bias[e]);
    write8<T, CODES>(g, row, c, y);
  }, end);
}

// ---- backward -----------------------------------------------------------------------------
//
// A group of rows per workgroup (per wave where a row is one wave's): its threads keep their columns,
// whose sums for dg and db stay in registers over the group's rows, and the groups' sums are added by a
// second launch. A row's x and dy are read one row ahead.
// Bound: HBM, x and dy read and dx written, and 8 bytes a column for each group: 8192 x 4096 bfloat16
// 39 us (5.1 TB/s without the groups' sums), the second launch's 4 among them, float32 80.
struct GradArgs {
  const void *x, *dy;
  int64_t x_ld, dy_ld, rows, cols;
  const void* weight;
  int32_t w_elem;
  const float *mean, *rstd;
  void* dx;        // [rows][cols], or null
  float *dg, *db;  // [groups][cols] each, or null
};

template <typename T, int LANES, int K>
__global__ __launch_bounds__(threads_of(LANES)) void norm_grad_kernel(GradArgs g) {
  constexpr int kEach = threads_of(LANES) / LANES;  // rows at a time
  constexpr int kWaves = LANES > kWave ? LANES / kWave : 1;
  __shared__ float sums[2][2][kWaves];
  __shared__ float join[kEach > 1 ? kEach * LANES * 8 : 1];
  const int lane = threadIdx.x % LANES, y = threadIdx.x / LANES;
  const int64_t groups = (int64_t)gridDim.x * kEach, group = (int64_t)blockIdx.x * kEach + y;
  const float scale = 1.f / (float)g.cols;
  float dg[K][8], db[K][8], gain[K][8];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int64_t c = 8 * (lane + k * LANES);
    parameters8(g.weight, g.w_elem, c, g.cols - c, 1.f, gain[k]);
#pragma unroll
    for (int e = 0; e < 8; ++e) dg[k][e] = db[k][e] = 0.f;
  }
  struct Row {
    Square<T> x, dy;  // K of their rows
    float mean, rstd;
  };
  auto read = [&](Row& r, int64_t row) {
    const T* x = reinterpret_cast<const T*>(g.x) + row * g.x_ld;
    const T* dy = reinterpret_cast<const T*>(g.dy) + row * g.dy_ld;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int64_t c = 8 * (lane + k * LANES);
      if (c + 8 <= g.cols) {
        r.x.load(k, x + c);
        r.dy.load(k, dy + c);
      } else {
        r.x.load(k, x + c, g.cols - c);
        r.dy.load(k, dy + c, g.cols - c);
      }
    }
    r.mean = g.mean[row];
    r.rstd = g.rstd[row];
  };
  auto take = [&](const Row& r, int64_t row, int parity) {
    float a = 0.f, b = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int64_t c = 8 * (lane + k * LANES);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        // Past the last column dy is zero, but mean / deviation may be an infinity.
        const float u = c + e < g.cols ? (r.x.value(k, e) - r.mean) * r.rstd : 0.f;
        const float d = r.dy.value(k, e), w = d * gain[k][e];
        a += w;
        b = __builtin_fmaf(w, u, b);
        dg[k][e] = __builtin_fmaf(d, u, dg[k][e]);
        db[k][e] += d;
      }
    }
    if (!g.dx) return;
#pragma unroll
    for (int off = (LANES < kWave ? LANES : kWave) / 2; off >= 1; off >>= 1) {
      a += __shfl_xor(a, off, kWave);
      b += __shfl_xor(b, off, kWave);
    }
    if constexpr (LANES > kWave) {
      if ((threadIdx.x & 63) == 0) {
        sums[parity][0][threadIdx.x >> 6] = a;
        sums[parity][1][threadIdx.x >> 6] = b;
      }
      __syncthreads();
      a = b = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        a += sums[parity][0][w];
        b += sums[parity][1][w];
      }
    }
    a *= scale;
    b *= scale;
    T* dx = reinterpret_cast<T*>(g.dx) + row * g.cols;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int64_t c = 8 * (lane + k * LANES);
      if (c >= g.cols) continue;
      float o[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {  // past the last column: not stored
        const float u = (r.x.value(k, e) - r.mean) * r.rstd;
        o[e] = ((r.dy.value(k, e) * gain[k][e] - a) - u * b) * r.rstd;
      }
      store8<T>(dx + c, o, g.cols - c);
    }
  };
  // Two rows' registers in turn. Every thread of a workgroup takes the same number of rows where rows
  // are more than a wave's (kEach is 1 then), so that all of them meet at the barriers.
  Row p, q;
  int64_t row = group;
  if (row < g.rows) read(p, row);
  for (; row < g.rows; row += 2 * groups) {
    if (row + groups < g.rows) read(q, row + groups);
    take(p, row, 0);
    if (row + groups >= g.rows) break;
    if (row + 2 * groups < g.rows) read(p, row + 2 * groups);
    take(q, row + groups, 1);
  }
  auto write = [&](float (&v)[K][8], float* to) {
    if (!to) return;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int64_t c = 8 * (lane + k * LANES);
      if constexpr (kEach > 1) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 8; ++e) join[(y * 8 + e) * LANES + lane] = v[k][e];
        __syncthreads();
        if (y == 0) {
#pragma unroll
          for (int i = 1; i < kEach; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[k][e] += join[(i * 8 + e) * LANES + lane];
        }
      }
      if (y == 0 && c < g.cols) store8<float>(to + blockIdx.x * g.cols + c, v[k], g.cols - c);
    }
  };
  write(dg, g.dg);
  write(db, g.db);
}

// Rows past the registers: a workgroup a row for dx, which reads x and dy twice; the column sums read them
// again. dx, column sums and their join, us: 2048 x 12288 bfloat16 33 + 16 + 4, 2048 x 16384 44 + 25 + 4 (float32 99 +
// 55 + 5), 2048 x 20000 58 + 28 + 5: 2.7 TB/s of the 201 MB that 2048 x 16384 has to read and write, where rows of
// 8192 columns, read once, take 24 + 4 for half of it.
template <typename T>
__global__ __launch_bounds__(kWide) void norm_grad_wide_kernel(GradArgs g) {
  __shared__ float sums[2][kWide / kWave];
  const int64_t row = blockIdx.x;
  const T* x = reinterpret_cast<const T*>(g.x) + row * g.x_ld;
  const T* dy = reinterpret_cast<const T*>(g.dy) + row * g.dy_ld;
  const float mean = g.mean[row], rstd = g.rstd[row], scale = 1.f / (float)g.cols;
  float a = 0.f, b = 0.f;
  for (int64_t c = 8 * threadIdx.x; c < g.cols; c += 8 * kWide) {
    float v[8], d[8], gain[8], pa = 0.f, pb = 0.f;
    values8<T>(x, c, g.cols - c, v);
    values8<T>(dy, c, g.cols - c, d);
    parameters8(g.weight, g.w_elem, c, g.cols - c, 1.f, gain);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float w = d[e] * gain[e], u = c + e < g.cols ? (v[e] - mean) * rstd : 0.f;
      pa += w;
      pb = __builtin_fmaf(w, u, pb);
    }
    a += pa;
    b += pb;
  }
  a = row_sum<kWide>(a, sums[0]) * scale;
  b = row_sum<kWide>(b, sums[1]) * scale;
  for (int64_t c = 8 * threadIdx.x; c < g.cols; c += 8 * kWide) {
    float v[8], d[8], gain[8], o[8];
    values8<T>(x, c, g.cols - c, v);
    values8<T>(dy, c, g.cols - c, d);
    parameters8(g.weight, g.w_elem, c, g.cols - c, 1.f, gain);
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = ((d[e] * gain[e] - a) - (v[e] - mean) * rstd * b) * rstd;
    store8<T>(reinterpret_cast<T*>(g.dx) + row * g.cols + c, o, g.cols - c);
  }
}

// The same rows' column sums: 256 columns and a range of rows a workgroup.
template <typename T>
__global__ __launch_bounds__(256) void norm_columns_kernel(GradArgs g, int64_t per) {
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= g.cols) return;
  const T* x = reinterpret_cast<const T*>(g.x) + c;
  const T* dy = reinterpret_cast<const T*>(g.dy) + c;
  const int64_t first = blockIdx.y * per, last = min(first + per, g.rows);
  float s = 0.f, t = 0.f;
#pragma unroll 4
  for (int64_t r = first; r < last; ++r) {
    const float d = (float)dy[r * g.dy_ld];
    s = __builtin_fmaf(d, ((float)x[r * g.x_ld] - g.mean[r]) * g.rstd[r], s);
    t += d;
  }
  if (g.dg) g.dg[blockIdx.y * g.cols + c] = s;
  if (g.db) g.db[blockIdx.y * g.cols + c] = t;
}

// dg and db: the groups' sums, 16 waves a column's, each every 16th in order.
struct JoinArgs {
  const float* parts[2];
  void* out[2];
  int32_t elem[2];
  int64_t count, cols;
};
__global__ __launch_bounds__(1024) void norm_join_kernel(JoinArgs g) {
  __shared__ float sums[16][kWave];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, which = blockIdx.y;
  const int64_t c = (int64_t)blockIdx.x * kWave + lane;
  if (!g.out[which]) return;
  const float* parts = g.parts[which] + c;
  float s = 0.f;
  if (c < g.cols)
#pragma unroll 8
    for (int64_t i = w; i < g.count; i += 16) s += parts[i * g.cols];
  sums[w][lane] = s;
  __syncthreads();
  if (w || c >= g.cols) return;
  float t = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) t += sums[i][lane];
  if (g.elem[which] == kF32) static_cast<float*>(g.out[which])[c] = t;
  else if (g.elem[which] == kBF16) static_cast<__bf16*>(g.out[which])[c] = (__bf16)t;
  else static_cast<_Float16*>(g.out[which])[c] = (_Float16)t;
}

// ---- launches -----------------------------------------------------------------------------

// A launch takes fewer than 2^32 threads.
bool fits(int64_t groups, int threads) { return groups <= (int64_t)UINT32_MAX / threads; }

template <typename T, int LANES, int K, bool CODES>
int launch_norm(const NormArgs& g, hipStream_t stream) {
  constexpr int threads = threads_of(LANES);
  const int64_t grid = ceil_div(g.rows, threads / LANES);
  DIONW_REQUIRE(fits(grid, threads), "layer_norm: too many rows");
  hipLaunchKernelGGL((norm_kernel<T, LANES, K, CODES>), dim3((unsigned)grid), dim3(threads), 0, stream, g);
  return check_launch("layer_norm");
}

// Fewer threads a row wait less for each other, more of them hold more rows' loads in flight. us of
// 64 2 / 64 4 / 128 2 / 256 1 / 256 2 / 512 1, bfloat16: 8192 x 768 7.7 / 9.8 / 9.9 / 12.0 / 14.8 / 22.0, 16384 x
// 2048 - / 25.0 / 22.9 / 27.3 / 27.8 / 42.4, 8192 x 4096 (64 8 28.6, 128 4 24.7) 256 2 23.3, 512 1 26.7.
template <typename T, bool CODES>
int launch_norm(const NormArgs& g, hipStream_t stream) {
  if (g.cols <= 128 && !CODES) return launch_norm<T, 16, 1, false>(g, stream);
  if (g.cols <= 512) return launch_norm<T, 64, 1, CODES>(g, stream);
  if (g.cols <= 1024) return launch_norm<T, 64, 2, CODES>(g, stream);
  if (g.cols <= 2048) return launch_norm<T, 128, 2, CODES>(g, stream);
  if (g.cols <= 4096) return launch_norm<T, 256, 2, CODES>(g, stream);
  if (g.cols <= 8192) return launch_norm<T, 256, 4, CODES>(g, stream);
  if (g.cols <= 16384) return launch_norm<T, 512, 4, CODES>(g, stream);
  hipLaunchKernelGGL((norm_wide_kernel<T, CODES>), dim3((unsigned)g.rows), dim3(kWide), 0, stream, g);
  return check_launch("layer_norm_wide");
}

template <bool CODES>
int launch_norm(int32_t elem, const NormArgs& g, hipStream_t stream) {
  if (elem == kF16) return launch_norm<_Float16, CODES>(g, stream);
  if (elem == kBF16) return launch_norm<__bf16, CODES>(g, stream);
  return launch_norm<float, CODES>(g, stream);
}

constexpr int64_t kWidest = 8192;  // columns of a row whose gradients a workgroup's registers hold

// Groups of rows whose column sums are kept apart: as many as run at a time, of two rows a wave or
// workgroup at least. us, bfloat16, 256 / 512 / 768 / 1024 groups: 8192 x 4096 42 / 39.3 / 46 / 46, 16384 x
// 2048 - / 41 / 38 / 40, 8192 x 768 20 / 16.3 / 20.6 / 21, 32768 x 300 55 / 34 / 30 / 28, 2048 x 1024 9.5 / 10.6.
int64_t row_groups(int64_t rows, int64_t cols) {
  if (cols > kWidest) return std::min<int64_t>(64, rows);
  const int each = cols <= 1024 ? 8 : 2;
  return std::min<int64_t>(ceil_div(rows, each), cols <= 512 ? 1024 : cols <= 4096 ? 512 : 256);
}

template <typename T, int LANES, int K>
int launch_grad(const GradArgs& g, hipStream_t stream) {
  constexpr int threads = threads_of(LANES);
  hipLaunchKernelGGL((norm_grad_kernel<T, LANES, K>), dim3((unsigned)row_groups(g.rows, g.cols)), dim3(threads), 0,
                     stream, g);
  return check_launch("layer_norm_backward");
}

template <typename T>
int launch_grad(const GradArgs& g, hipStream_t stream) {
  if (g.cols <= 512) return launch_grad<T, 64, 1>(g, stream);
  if (g.cols <= 1024) return launch_grad<T, 64, 2>(g, stream);
  if (g.cols <= 2048) return launch_grad<T, 256, 1>(g, stream);
  if (g.cols <= 4096) return launch_grad<T, 256, 2>(g, stream);
  if (g.cols <= kWidest) return launch_grad<T, 512, 2>(g, stream);
  if (g.dx) {
    hipLaunchKernelGGL(norm_grad_wide_kernel<T>, dim3((unsigned)g.rows), dim3(kWide), 0, stream, g);
    DIONW_TRY(check_launch("layer_norm_backward_wide"));
  }
  if (!g.dg && !g.db) return kOk;
  const int64_t groups = row_groups(g.rows, g.cols);
  hipLaunchKernelGGL(norm_columns_kernel<T>, dim3((unsigned)ceil_div(g.cols, 256), (unsigned)groups), dim3(256), 0,
                     stream, g, ceil_div(g.rows, groups));
  return check_launch("layer_norm_columns");
}

bool good_elem(int32_t e) { return e == kF16 || e == kBF16 || e == kF32; }

int check_norm(int32_t elem, const void* x, int64_t x_ld, int64_t rows, int64_t cols, int32_t w_elem,
               int32_t b_elem) {
  DIONW_REQUIRE(good_elem(elem) && good_elem(w_elem) && good_elem(b_elem), "layer_norm: bad element type");
  DIONW_REQUIRE(rows >= 0 && cols > 0 && cols < INT32_MAX / 2, "layer_norm: bad extents %lld x %lld",
                (long long)rows, (long long)cols);
  DIONW_REQUIRE(rows == 0 || (x && x_ld >= cols), "layer_norm: bad input");
  // As many as their gradients' kernel takes too.
  DIONW_REQUIRE(cols <= kWidest || fits(rows, kWide), "layer_norm: too many rows");
  return kOk;
}

}  // namespace
}  // namespace dionw

using namespace dionw;

extern "C" {

int dionw_layer_norm_forward(int32_t elem, const void* x, int64_t x_ld, int64_t rows, int64_t cols,
                             int32_t w_elem, const void* weight, int32_t b_elem, const void* bias,
                             float eps, void* y, float* mean, float* rstd, hipStream_t stream) {
  DIONW_TRY(check_norm(elem, x, x_ld, rows, cols, w_elem, b_elem));
  if (rows == 0) return kOk;
  DIONW_REQUIRE(y && !mean == !rstd, "layer_norm: bad output");
  NormArgs g{};
  g.x = x;
  g.x_ld = x_ld;
  g.rows = rows;
  g.cols = cols;
  g.weight = weight;
  g.bias = bias;
  g.w_elem = w_elem;
  g.b_elem = b_elem;
  g.eps = eps;
  g.y = y;
  g.mean = mean;
  g.rstd = rstd;
  return launch_norm<false>(elem, g, stream);
}

int dionw_layer_norm_float4(int32_t elem, const void* x, int64_t x_ld, int64_t rows, int64_t cols,
                            int32_t w_elem, const void* weight, int32_t b_elem, const void* bias,
                            float eps, void* data, void* scale, int64_t scale_ld, hipStream_t stream) {
  DIONW_TRY(check_norm(elem, x, x_ld, rows, cols, w_elem, b_elem));
  if (rows == 0) return kOk;
  DIONW_REQUIRE(data && scale && aligned16(data) && scale_ld >= rows, "layer_norm: bad output");
  NormArgs g{};
  g.x = x;
  g.x_ld = x_ld;
  g.rows = rows;
  g.cols = cols;
  g.weight = weight;
  g.bias = bias;
  g.w_elem = w_elem;
  g.b_elem = b_elem;
  g.eps = eps;
  g.data = static_cast<uint8_t*>(data);
  g.scale = static_cast<uint8_t*>(scale);
  g.depth = round_up(cols, kDepth4);
  g.scale_ld = scale_ld;
  return launch_norm<true>(elem, g, stream);
}

size_t dionw_layer_norm_backward_scratch(int64_t rows, int64_t cols) {
  return rows > 0 && cols > 0 ? (size_t)(2 * row_groups(rows, cols) * cols) * sizeof(float) : 0;
}

int dionw_layer_norm_backward(int32_t elem, const void* x, int64_t x_ld, const void* dy, int64_t dy_ld,
                              int64_t rows, int64_t cols, int32_t w_elem, const void* weight,
                              const float* mean, const float* rstd, void* dx, void* dg,
                              int32_t b_elem, void* db, void* scratch, size_t scratch_bytes,
                              hipStream_t stream) {
  DIONW_TRY(check_norm(elem, x, x_ld, rows, cols, w_elem, b_elem));
  DIONW_REQUIRE(rows == 0 || (dy && dy_ld >= cols && mean && rstd), "layer_norm: bad input");
  const size_t need = dg || db ? dionw_layer_norm_backward_scratch(rows, cols) : 0;
  DIONW_REQUIRE(need == 0 || (scratch && scratch_bytes >= need && (reinterpret_cast<uintptr_t>(scratch) & 3) == 0),
                "layer_norm: scratch too small");
  const int64_t groups = rows ? row_groups(rows, cols) : 0;
  float* parts = static_cast<float*>(scratch);
  const GradArgs g{x, dy, x_ld, dy_ld, rows, cols, weight, w_elem, mean, rstd, dx,
                   dg ? parts : nullptr, db ? parts + groups * cols : nullptr};
  if (rows && (dx || dg || db)) {
    if (elem == kF16) DIONW_TRY(launch_grad<_Float16>(g, stream));
    if (elem == kBF16) DIONW_TRY(launch_grad<__bf16>(g, stream));
    if (elem == kF32) DIONW_TRY(launch_grad<float>(g, stream));
  }
  if (!dg && !db) return kOk;
  const JoinArgs j{{g.dg, g.db}, {dg, db}, {w_elem, b_elem}, groups, cols};
  hipLaunchKernelGGL(norm_join_kernel, dim3((unsigned)ceil_div(cols, kWave), 2), dim3(1024), 0, stream, j);
  return check_launch("layer_norm_join");
}

}  // extern "C"

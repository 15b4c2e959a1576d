// RMS norm with the residual's addition, its gradients, and values in 8 bits with a scale for each block of 128 columns.
//
//   h = round(x + residual)     n = 1 / sqrt(mean(h^2) + eps)     y = h n w
//   dh = dsum + n (w dy - h n^2 mean(w dy h))     dw = sum over rows of dy h n
//
// The norm is that of the sum as its type holds it: what the next layers read is what was normalised, and the backward
// pass needs nothing but that sum.  Statistics and products are in 32 bits, each output is rounded once.
#include "rows.hpp"

#include <algorithm>
#include <type_traits>

namespace mv {
namespace {

constexpr int kThreads = 256;
constexpr int kMostColumns = 16384;   // of a row in registers

template <typename V> __device__ __forceinline__ V wave_sum(V v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
  return v;
}
// Sum over the workgroup, the same for every thread.
template <int Threads = kThreads, typename V> __device__ __forceinline__ V block_sum(V v, V *lds) {
  v = wave_sum(v);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int i = 0; i < Threads / 64; ++i) v += lds[i];
  __syncthreads();
  return v;
}

// Sum of eight products, in pairs.
__device__ __forceinline__ float dot8(const float (&a)[8], const float (&b)[8]) {
  float s[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) s[i] = fmaf(a[i], b[i], a[i + 4] * b[i + 4]);
  return (s[0] + s[1]) + (s[2] + s[3]);
}

// 1 / sqrt(a) to the last bit but one: the hardware's value (1 ulp), corrected by what a r^2 is off from 1, in two parts.
__device__ __forceinline__ float inverse_root(float a) {
  const float r = __builtin_amdgcn_rsqf(a), t = a * r, rest = fmaf(a, r, -t);
  const float e = fmaf(-t, r, 1.f) - rest * r, better = fmaf(0.5f * r, e, r);
  return better == better ? better : r;   // (0, infinity, NaN, and numbers so small that a r is none)
}

// 1 / sqrt(a) of a row in two parts, corrected in the same way: results in front of a scale of 8-bit values are then off by their
// own roundings alone (16-bit rows, 55296 x 1000 in 8 bits: 74 -> 75 us).  float32 rows sum their squares over lanes in 64
// bits too, memory leaves the time for it; 16-bit rows would take 78 us with that.
template <typename T> using SumOf = std::conditional_t<sizeof(T) == 4, double, float>;
struct Root {
  float high, low = 0.f;
  __device__ __forceinline__ explicit Root(float a) {
    const float r = __builtin_amdgcn_rsqf(a), t = a * r, rest = fmaf(a, r, -t);
    const float step = 0.5f * r * (fmaf(-t, r, 1.f) - rest * r);
    high = r + step, low = (r - high) + step;
    if (high != high) high = r;   // (0, infinity, NaN, and numbers so small that a r is none)
    if (low != low) low = 0.f;
  }
  __device__ __forceinline__ explicit Root(double a) {
    double r = __builtin_amdgcn_rsq(a);
    const double better = fma(0.5 * r, fma(-a * r, r, 1.), r);
    if (better == better) r = better;   // (0, infinity, NaN)
    high = static_cast<float>(r), low = static_cast<float>(r - high);
    if (low != low) low = 0.f;
  }
};

// v w n: 16-bit factors v, w have an exact product (16-bit rows with float32 weights: to 2^-24); of others the rest goes into the
// second one.
template <typename T> __device__ __forceinline__ float scaled(float v, float w, const Root &n) {
  const float p = v * w;
  const float most = fmaf(p, n.high, sizeof(T) == 2 ? p * n.low : fmaf(p, n.low, fmaf(v, w, -p) * n.high));
  return most == most ? most : p * n.high;   // (an infinite product has no rest)
}

__device__ __forceinline__ void load_weight(const void *w, bool wide, const float *, int col, int left, float (&out)[8]) {
  load8(static_cast<const float *>(w) + col, left, out);
}
template <typename T>
__device__ __forceinline__ void load_weight(const void *w, bool wide, const T *, int col, int left, float (&out)[8]) {
  if (wide) load8(static_cast<const float *>(w) + col, left, out);
  else load8(static_cast<const T *>(w) + col, left, out);
}

// The scale of 128 columns that 16 neighbouring lanes hold, eight each.
__device__ __forceinline__ float lanes_scale(const float (&v)[8]) {
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) most = max_abs(most, v[i]);
#pragma unroll
  for (int d = 8; d; d >>= 1) most = max_abs(most, __shfl_xor(most, d));
  return block_scale(most);
}

// Sum over the Lanes threads of a row, the same for each of them
template <int Lanes, typename V> __device__ __forceinline__ V row_sum(V v, V *lds) {
  if constexpr (Lanes >= kThreads) return block_sum<Lanes>(v, lds);
  if constexpr (Lanes == 128) {   // two wavefronts
    v = wave_sum(v);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = lds[threadIdx.x / 128 * 2] + lds[threadIdx.x / 128 * 2 + 1];
    __syncthreads();
    return v;
  }
#pragma unroll
  for (int d = Lanes / 2; d; d >>= 1) v += __shfl_xor(v, d);
  return v;
}

constexpr int threads_of(int lanes) { return lanes > kThreads ? lanes : kThreads; }

// Rows that fit into registers: Lanes threads, 8 Chunks columns each.  One pass over memory, which bounds it: 55296 x 256 in
// bf16 with residual 19 us (5.9 TB/s for four bytes in and four out of an element), 55296 x 1000 78 us (5.6 TB/s), in 8 bits
// 75 us (5.2 TB/s).  Rows of 1003 columns start at any byte: 97 us.  A wavefront or less takes a row as long as there
// are 512 columns (no barrier); 513 to 1024 columns run on two wavefronts with eight columns per thread (on one with sixteen,
// the gradients below took 150 instead of 105 us: half as many loads in flight), more than 4096 on 512 or 1024 threads with
// sixteen (5000 x 8192 61 us; with 32 on 256 threads 65).  10000 columns 62 us of 4000 rows (72 in two passes).
template <typename T, int Lanes, int Chunks>
__global__ __launch_bounds__(threads_of(Lanes)) void norm_rows(const T *x, const T *residual, const void *weight, bool wide, T *y, unsigned char *q,
                                                      float *scales, T *sum, long rows, int columns, float eps) {
  __shared__ SumOf<T> lds[threads_of(Lanes) / 64];
  const long mine = static_cast<long>(linear_block()) * (threads_of(Lanes) / Lanes) + threadIdx.x / Lanes;
  if (mine >= rows && (Lanes != 128 || mine - threadIdx.x / Lanes >= rows)) return;   // (two rows wait for each other)
  const long row = min(mine, rows - 1);   // (the last one twice, with the same results)
  const int lane = threadIdx.x % Lanes;
  const long at = row * columns;
  float v[Chunks][8], squares = 0.f;
#pragma unroll
  for (int k = 0; k < Chunks; ++k) {
    const int c = (k * Lanes + lane) * 8;
    load8(x + at + c, columns - c, v[k]);
  }
  if (residual) {
    float r[Chunks][8];
#pragma unroll
    for (int k = 0; k < Chunks; ++k) {
      const int c = (k * Lanes + lane) * 8;
      load8(residual + at + c, columns - c, r[k]);
    }
#pragma unroll
    for (int k = 0; k < Chunks; ++k) {
      const int c = (k * Lanes + lane) * 8;
#pragma unroll
      for (int i = 0; i < 8; ++i) v[k][i] += r[k][i];
      if constexpr (sizeof(T) == 2) {   // what is stored is what is normalised
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const unsigned both = pack2<T>(v[k][2 * i], v[k][2 * i + 1]);
          v[k][2 * i] = Bits<T>::up(static_cast<unsigned short>(both & 0xffffu));
          v[k][2 * i + 1] = Bits<T>::up(static_cast<unsigned short>(both >> 16));
        }
      }
      store8(sum + at + c, columns - c, v[k]);
    }
  }
#pragma unroll
  for (int k = 0; k < Chunks; ++k) squares += dot8(v[k], v[k]);
  const Root n(row_sum<Lanes>(static_cast<SumOf<T>>(squares), lds) / columns + eps);
  const int padded = (columns + kBlock - 1) / kBlock * kBlock;
#pragma unroll
  for (int k = 0; k < Chunks; ++k) {
    const int c = (k * Lanes + lane) * 8;
    float w[8];
    load_weight(weight, wide, x, c, columns - c, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[k][i] = scaled<T>(v[k][i], w[i], n);
    if (!q) {
      store8(y + at + c, columns - c, v[k]);
      continue;
    }
    const float s = lanes_scale(v[k]), inverse = 1.f / s;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[k][i] *= inverse;
    if (c < padded) {
      *reinterpret_cast<u32x2 *>(q + row * padded + c) = to_e4m3(v[k]);
      if ((lane & 15) == 0) scales[row * (padded / kBlock) + c / kBlock] = s;
    }
  }
}

// Both gradients in one pass over memory: a workgroup takes every gridDim-th row (or group of rows), and keeps its share of
// the weight's gradient in registers until the end.  Bound by memory: 55296 x 256 in bf16 with both incoming gradients 29 us
// (3.9 TB/s), 55296 x 1000 100 us (4.4 TB/s), with the join of 1024 partial sums (1536: 32 and 125 us, 512: 35 and 164); float32
// 6000 x 4096 82 us (4.8 TB/s) and 7 for the join.
// Longer rows have fewer workgroups, and as many fewer partial sums: 5000 x 8192 on 512 of 512 threads 76 us (115 on 1024 of
// 256, 108 on 512 of those); beyond 8192 columns on 512 threads with 32 columns each (3000 x 16384 127 us; two passes 164, 1024
// threads with sixteen spill 275 registers: 338).
template <typename T, int Lanes, int Chunks>
__global__ __launch_bounds__(threads_of(Lanes)) void norm_grad(const T *h, const void *weight, bool wide, const T *gy, const T *gsum, T *gx,
                                                      float *partial, long rows, int columns, float eps) {
  constexpr int kGroups = threads_of(Lanes) / Lanes;
  __shared__ float lds[threads_of(Lanes) / 64];
  __shared__ float sums[kGroups > 1 ? kGroups - 1 : 1][Lanes * Chunks * 8];
  const int lane = threadIdx.x % Lanes, group = threadIdx.x / Lanes;
  float w[Chunks][8], dw[Chunks][8] = {};
#pragma unroll
  for (int k = 0; k < Chunks; ++k) {
    const int c = (k * Lanes + lane) * 8;
    load_weight(weight, wide, h, c, columns - c, w[k]);
  }
  for (long first = static_cast<long>(blockIdx.x) * kGroups; first < rows; first += static_cast<long>(gridDim.x) * kGroups) {
    const long row = min(first + group, rows - 1), at = row * columns;
    const bool live = first + group < rows;
    float v[Chunks][8], g[Chunks][8], s[Chunks][8], squares = 0.f, dot = 0.f;
#pragma unroll
    for (int k = 0; k < Chunks; ++k) {
      const int c = (k * Lanes + lane) * 8, left = live ? columns - c : 0;
      load8(h + at + c, left, v[k]);
      load8(gy + at + c, left, g[k]);
      if (gsum) load8(gsum + at + c, left, s[k]);
    }
#pragma unroll
    for (int k = 0; k < Chunks; ++k) {
      float gw[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) gw[i] = g[k][i] * w[k][i];
      squares += dot8(v[k], v[k]);
      dot += dot8(gw, v[k]);
    }
    const float n = inverse_root(row_sum<Lanes>(squares, lds) / columns + eps);
    const float back = row_sum<Lanes>(dot, lds) / columns * n * n;
#pragma unroll
    for (int k = 0; k < Chunks; ++k) {
      const int c = (k * Lanes + lane) * 8;
      float d[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        d[i] = n * (g[k][i] * w[k][i] - v[k][i] * back) + (gsum ? s[k][i] : 0.f);
        dw[k][i] += live ? g[k][i] * (v[k][i] * n) : 0.f;
      }
      if (live && gx) store8(gx + at + c, columns - c, d);
    }
  }
  if (!partial) return;
  if constexpr (kGroups > 1) {   // the groups' shares, in their order
    if (group) {
#pragma unroll
      for (int k = 0; k < Chunks; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) sums[group - 1][(k * Lanes + lane) * 8 + i] = dw[k][i];
    }
    __syncthreads();
    if (group) return;
    for (int o = 0; o < kGroups - 1; ++o)
#pragma unroll
      for (int k = 0; k < Chunks; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) dw[k][i] += sums[o][(k * Lanes + lane) * 8 + i];
  }
#pragma unroll
  for (int k = 0; k < Chunks; ++k) {
    const int c = (k * Lanes + lane) * 8;
    store8(partial + static_cast<long>(blockIdx.x) * columns + c, columns - c, dw[k]);
  }
}

// ---- rows of any length ------------------------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(kThreads) void norm_long_rows(const T *x, const T *residual, const void *weight, bool wide, T *y,
                                                        unsigned char *q, float *scales, T *sum, long rows, int columns,
                                                        float eps) {
  __shared__ SumOf<T> lds[kThreads / 64];
  const long row = linear_block();
  if (row >= rows) return;
  const T *xr = x + row * columns;
  SumOf<T> squares = 0;
  for (int c = threadIdx.x * 8; c < columns; c += kThreads * 8) {
    float v[8], r[8];
    load8(xr + c, columns - c, v);
    if (residual) {
      load8(residual + row * columns + c, columns - c, r);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = load(&(const T &)store_cast<T>(v[i] + r[i]));
      store8(sum + row * columns + c, columns - c, v);
    }
    squares += dot8(v, v);
  }
  const Root n(block_sum(squares, lds) / columns + eps);
  const T *hr = residual ? sum + row * columns : xr;
  const int padded = (columns + kBlock - 1) / kBlock * kBlock;
  for (int c = threadIdx.x * 8; c < (q ? padded : columns); c += kThreads * 8) {
    float v[8], w[8];
    load8(hr + c, columns - c, v);
    load_weight(weight, wide, x, c, columns - c, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = scaled<T>(v[i], w[i], n);
    if (!q) {
      store8(y + row * columns + c, columns - c, v);
      continue;
    }
    const float s = lanes_scale(v), inverse = 1.f / s;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= inverse;
    *reinterpret_cast<u32x2 *>(q + row * padded + c) = to_e4m3(v);
    if ((threadIdx.x & 15) == 0) scales[row * (padded / kBlock) + c / kBlock] = s;
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void norm_grad_long_rows(const T *h, const void *weight, bool wide, const T *gy, const T *gsum,
                                                           T *gx, float *norms, long rows, int columns, float eps) {
  __shared__ float lds[kThreads / 64];
  const long row = linear_block();
  if (row >= rows) return;
  float squares = 0.f, dot = 0.f;
  for (int c = threadIdx.x * 8; c < columns; c += kThreads * 8) {
    float v[8], g[8], w[8];
    load8(h + row * columns + c, columns - c, v);
    load8(gy + row * columns + c, columns - c, g);
    load_weight(weight, wide, h, c, columns - c, w);
    squares += dot8(v, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) g[i] *= w[i];
    dot += dot8(g, v);
  }
  const float n = inverse_root(block_sum(squares, lds) / columns + eps);
  const float back = block_sum(dot, lds) / columns * n * n;
  if (threadIdx.x == 0 && norms) norms[row] = n;
  if (!gx) return;
  for (int c = threadIdx.x * 8; c < columns; c += kThreads * 8) {
    float v[8], g[8], w[8], s[8];
    load8(h + row * columns + c, columns - c, v);
    load8(gy + row * columns + c, columns - c, g);
    load_weight(weight, wide, h, c, columns - c, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = n * (g[i] * w[i] - v[i] * back);
    if (gsum) {
      load8(gsum + row * columns + c, columns - c, s);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] += s[i];
    }
    store8(gx + row * columns + c, columns - c, v);
  }
}

constexpr int kSlices = 64;   // of the rows, for the gradient of the weight

// Thread = eight columns of one slice of rows.
template <typename T>
__global__ __launch_bounds__(kThreads) void norm_grad_long_columns(const T *h, const T *gy, const float *norms, float *partial,
                                                              long rows, int columns) {
  const int c = (blockIdx.x * kThreads + threadIdx.x) * 8;
  if (c >= columns) return;
  const long each = (rows + kSlices - 1) / kSlices, first = blockIdx.y * each, last = min(rows, first + each);
  float sum[8] = {};
  for (long row = first; row < last; ++row) {
    float v[8], g[8];
    load8(h + row * columns + c, columns - c, v);
    load8(gy + row * columns + c, columns - c, g);
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[i] += g[i] * (v[i] * norms[row]);
  }
  store8(partial + static_cast<long>(blockIdx.y) * columns + c, columns - c, sum);
}

// Sum of the partial sums, in a fixed order: 16 columns and 16 shares of the parts per workgroup
template <typename T>
__global__ __launch_bounds__(kThreads) void norm_grad_weight(const float *partial, void *gw, bool wide, int columns, int parts) {
  __shared__ float sums[16][16];
  const int in = threadIdx.x & 15, share = threadIdx.x >> 4, c = blockIdx.x * 16 + in;
  float sum = 0.f;
  if (c < columns) {
#pragma unroll 8
    for (int p = share; p < parts; p += 16) sum += partial[static_cast<long>(p) * columns + c];
  }
  sums[share][in] = sum;
  __syncthreads();
  if (share || c >= columns) return;
  for (int i = 1; i < 16; ++i) sum += sums[i][in];
  if (wide) static_cast<float *>(gw)[c] = sum;
  else static_cast<T *>(gw)[c] = store_cast<T>(sum);
}

// 16 threads for a block of one row and 128 columns.  Bound by memory: 4000 x 12544 in bf16 33 us (150 MB, 4.6 TB/s);
// 8 x 87808, the first of two kernels of a call, 4 us.
constexpr int kAtOnce = 2;   // blocks of 16 threads, the loads of all before the first is used
template <typename T>
__global__ __launch_bounds__(kThreads) void quantize_rows(const T *x, unsigned char *q, float *scales, long blocks, int columns) {
  const int per_row = (columns + kBlock - 1) / kBlock;
  const long first = static_cast<long>(linear_block()) * (kAtOnce * kThreads / 16) + threadIdx.x / 16;
  if (first >= blocks) return;
  float v[kAtOnce][8];
  long row[kAtOnce];
  int c[kAtOnce];
#pragma unroll
  for (int n = 0; n < kAtOnce; ++n) {
    const long block = min(first + n * (kThreads / 16), blocks - 1);   // (beyond the last: that one again, with the same results)
    row[n] = blocks <= 0x7fffffff ? static_cast<unsigned>(block) / static_cast<unsigned>(per_row) : block / per_row;
    c[n] = static_cast<int>(block - row[n] * per_row) * kBlock + (threadIdx.x & 15) * 8;
    load8(x + row[n] * columns + c[n], columns - c[n], v[n]);
  }
#pragma unroll
  for (int n = 0; n < kAtOnce; ++n) {
    const float s = lanes_scale(v[n]), inverse = 1.f / s;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[n][i] *= inverse;
    *reinterpret_cast<u32x2 *>(q + row[n] * (static_cast<long>(per_row) * kBlock) + c[n]) = to_e4m3(v[n]);
    if ((threadIdx.x & 15) == 0) scales[row[n] * per_row + c[n] / kBlock] = s;
  }
}

// One workgroup for a block of 128 x 128: 16 rows at a time, twice (weights, once when a layer is built: 1024 x 87808 from
// float32 123 us).
template <typename T>
__global__ __launch_bounds__(kThreads) void quantize_tiles(const T *x, unsigned char *q, float *scales, long rows, int columns) {
  __shared__ float lds[kThreads / 64];
  const int per_row = (columns + kBlock - 1) / kBlock;
  const long tile = linear_block(), top = tile / per_row * kBlock;
  if (top >= rows) return;
  const int c = static_cast<int>(tile % per_row) * kBlock + (threadIdx.x & 15) * 8;
  float most = 0.f;
  for (long r = top + threadIdx.x / 16; r < min(rows, top + kBlock); r += kThreads / 16) {
    float v[8];
    load8(x + r * columns + c, columns - c, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) most = max_abs(most, v[i]);
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) most = max_abs(most, __shfl_xor(most, d));
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = most;
  __syncthreads();
  most = 0.f;
#pragma unroll
  for (int i = 0; i < kThreads / 64; ++i) most = max_abs(most, lds[i]);
  const float s = block_scale(most), inverse = 1.f / s;
  for (long r = top + threadIdx.x / 16; r < min(rows, top + kBlock); r += kThreads / 16) {
    float v[8];
    load8(x + r * columns + c, columns - c, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= inverse;
    *reinterpret_cast<u32x2 *>(q + r * (static_cast<long>(per_row) * kBlock) + c) = to_e4m3(v);
  }
  if (threadIdx.x == 0) scales[tile] = s;
}

// Calls f with the threads of a row and the pieces of eight columns of each, for rows of up to kMostColumns; false: longer
template <bool Gradients, typename F> bool for_row_shape(int columns, const F &f) {
  using std::integral_constant;
  if (columns <= 128) f(integral_constant<int, 16>(), integral_constant<int, 1>());
  else if (columns <= 256) f(integral_constant<int, 32>(), integral_constant<int, 1>());
  else if (columns <= 512) f(integral_constant<int, 64>(), integral_constant<int, 1>());
  else if (columns <= 1024) f(integral_constant<int, 128>(), integral_constant<int, 1>());
  else if (columns <= 2048) f(integral_constant<int, 256>(), integral_constant<int, 1>());
  else if (columns <= 4096) f(integral_constant<int, 256>(), integral_constant<int, 2>());
  else if (columns <= 8192) f(integral_constant<int, 512>(), integral_constant<int, 2>());
  else if (columns <= kMostColumns) f(integral_constant<int, Gradients ? 512 : 1024>(), integral_constant<int, Gradients ? 4 : 2>());
  return columns <= kMostColumns;
}

constexpr long kGradGroups = 1024;   // workgroups of 256 threads of the gradients' kernel: four per compute unit
// workgroups of it, and partial sums of the weight's gradient
int grad_parts(long rows, int columns) {
  const int per = columns <= 128 ? 16 : columns <= 256 ? 8 : columns <= 512 ? 4 : columns <= 1024 ? 2 : 1;
  const long most = columns <= 4096 ? kGradGroups : columns <= 8192 ? kGradGroups / 2 : kGradGroups / 4;
  return columns > kMostColumns ? kSlices : static_cast<int>(std::max(1L, std::min(most, (rows + per - 1) / per)));
}

int norm_arguments(long rows, int columns, int dtype, int weight_dtype) {
  MV_REQUIRE(dtype == MV_F32 || dtype == MV_F16 || dtype == MV_BF16, "dtype %d is not float32, float16 or bfloat16", dtype);
  MV_REQUIRE(weight_dtype == dtype || weight_dtype == MV_F32, "weight has dtype %d, expected %d or float32", weight_dtype, dtype);
  MV_REQUIRE(rows >= 0 && columns > 0 && columns <= (1 << 30), "wrong sizes: %ld rows of %d columns", rows, columns);
  return MV_OK;
}

int norm_forward(const void *x, const void *residual, const void *weight, void *y, void *q, void *scales, void *sum, long rows,
                 int columns, float eps, int dtype, int weight_dtype, void *stream) {
  if (const int status = norm_arguments(rows, columns, dtype, weight_dtype)) return status;
  if (rows == 0) return MV_OK;
  MV_REQUIRE(x && weight && (y || (q && scales)), "a tensor is missing");
  MV_REQUIRE(!residual == !sum, "the sum goes with a residual");
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const bool wide = weight_dtype == MV_F32;
  auto *const q8 = static_cast<unsigned char *>(q);
  auto *const sc = static_cast<float *>(scales);
  MV_FLOATS(dtype, {
    const T *const xt = static_cast<const T *>(x), *const rt = static_cast<const T *>(residual);
    T *const yt = static_cast<T *>(y), *const ht = static_cast<T *>(sum);
    const bool fits = for_row_shape<false>(columns, [&](auto lanes, auto chunks) {
      constexpr int kAll = threads_of(lanes), kRows = kAll / lanes;
      norm_rows<T, lanes, chunks><<<linear_grid((rows + kRows - 1) / kRows, kAll), kAll, 0, st>>>(xt, rt, weight, wide, yt, q8, sc, ht, rows, columns, eps);
    });
    if (!fits)
      norm_long_rows<T><<<linear_grid(rows, kThreads), kThreads, 0, st>>>(xt, rt, weight, wide, yt, q8, sc, ht, rows, columns, eps);
  })
  return check_launch("add_rms_norm");
}

}  // namespace
}  // namespace mv

using namespace mv;

extern "C" {

int mv_add_rms_norm(const void *x, const void *residual, const void *weight, void *y, void *sum, int64_t rows, int columns,
                    float eps, int dtype, int weight_dtype, void *stream) {
  return norm_forward(x, residual, weight, y, nullptr, nullptr, sum, rows, columns, eps, dtype, weight_dtype, stream);
}

int mv_add_rms_norm_quantized(const void *x, const void *residual, const void *weight, void *q, void *scales, void *sum,
                              int64_t rows, int columns, float eps, int dtype, int weight_dtype, void *stream) {
  return norm_forward(x, residual, weight, nullptr, q, scales, sum, rows, columns, eps, dtype, weight_dtype, stream);
}

size_t mv_add_rms_norm_backward_workspace_bytes(int64_t rows, int columns) {
  if (rows < 0 || columns <= 0) return 0;
  return 4 * ((columns > kMostColumns ? static_cast<size_t>(rows) : 0) + static_cast<size_t>(grad_parts(rows, columns)) * columns);
}

int mv_add_rms_norm_backward(const void *h, const void *weight, const void *grad_y, const void *grad_sum, void *grad_x,
                             void *grad_weight, int64_t rows, int columns, float eps, int dtype, int weight_dtype,
                             void *workspace, size_t workspace_bytes, void *stream) {
  if (const int status = norm_arguments(rows, columns, dtype, weight_dtype)) return status;
  if ((rows == 0 || !grad_x) && !grad_weight) return MV_OK;
  MV_REQUIRE(weight && (rows == 0 || (h && grad_y)), "a tensor is missing");
  MV_REQUIRE(!grad_weight || (workspace && workspace_bytes >= mv_add_rms_norm_backward_workspace_bytes(rows, columns)), "the workspace is too small");
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const bool wide = weight_dtype == MV_F32;
  const int parts = grad_parts(rows, columns);
  float *const partial = grad_weight ? static_cast<float *>(workspace) : nullptr;
  float *const norms = grad_weight ? partial + static_cast<long>(parts) * columns : nullptr;
  MV_FLOATS(dtype, {
    const T *const ht = static_cast<const T *>(h), *const gy = static_cast<const T *>(grad_y), *const gs = static_cast<const T *>(grad_sum);
    T *const gx = static_cast<T *>(grad_x);
    const bool fits = for_row_shape<true>(columns, [&](auto lanes, auto chunks) {
      norm_grad<T, lanes, chunks><<<parts, threads_of(lanes), 0, st>>>(ht, weight, wide, gy, gs, gx, partial, rows, columns, eps);
    });
    if (!fits) {
      if (rows > 0) norm_grad_long_rows<T><<<linear_grid(rows, kThreads), kThreads, 0, st>>>(ht, weight, wide, gy, gs, gx, norms, rows, columns, eps);
      if (grad_weight)
        norm_grad_long_columns<T><<<dim3((columns + kThreads * 8 - 1) / (kThreads * 8), kSlices), kThreads, 0, st>>>(ht, gy, norms, partial, rows, columns);
    }
    if (grad_weight) norm_grad_weight<T><<<(columns + 15) / 16, kThreads, 0, st>>>(partial, grad_weight, wide, columns, parts);
  })
  return check_launch("add_rms_norm backward");
}

int mv_quantize_blocks(const void *x, void *q, void *scales, int64_t rows, int columns, int block_rows, int dtype, void *stream) {
  MV_REQUIRE(block_rows == 1 || block_rows == kBlock, "block_rows %d: 1 or 128 are possible", block_rows);
  MV_REQUIRE(rows >= 0 && columns > 0 && columns <= (1 << 30), "wrong sizes: %ld rows of %d columns", static_cast<long>(rows), columns);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const long per_row = (columns + kBlock - 1) / kBlock;
  if (rows == 0) return MV_OK;
  MV_REQUIRE(x && q && scales, "a tensor is missing");
  MV_FLOATS(dtype, {
    if (block_rows == 1)
      quantize_rows<T><<<linear_grid((rows * per_row * 16 + kAtOnce * kThreads - 1) / (kAtOnce * kThreads), kThreads), kThreads, 0, s>>>(
          static_cast<const T *>(x), static_cast<unsigned char *>(q), static_cast<float *>(scales), rows * per_row, columns);
    else
      quantize_tiles<T><<<linear_grid((rows + kBlock - 1) / kBlock * per_row, kThreads), kThreads, 0, s>>>(
          static_cast<const T *>(x), static_cast<unsigned char *>(q), static_cast<float *>(scales), rows, columns);
  })
  return check_launch("quantize_blocks");
}

}  // extern "C"

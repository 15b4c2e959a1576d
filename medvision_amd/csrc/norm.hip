// RMS norm with the residual's addition, its gradients, and values in 8 bits with a scale for each block of 128 columns.
//
//   h = round(x + residual)     n = 1 / sqrt(mean(h^2) + eps)     y = h n w
//   dh = dsum + n (w dy - h n^2 mean(w dy h))     dw = sum over rows of dy h n
//
// The norm is that of the sum as its type holds it: what the next layers read is what was normalised, and the backward
// pass needs nothing but that sum.  Statistics and products are in 32 bits, each output is rounded once.
#include "rows.hpp"

namespace mv {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
  return v;
}
// Sum over the workgroup, the same for every thread.
__device__ __forceinline__ float block_sum(float v, float *lds) {
  v = wave_sum(v);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0.f;
#pragma unroll
  for (int i = 0; i < kThreads / 64; ++i) v += lds[i];
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

// v w n: 16-bit factors v, w have an exact product; of others the rest goes into the second one.
template <typename T> __device__ __forceinline__ float scaled(float v, float w, float n) {
  const float p = v * w;
  if constexpr (sizeof(T) == 2) return p * n;
  const float most = fmaf(p, n, fmaf(v, w, -p) * n);
  return most == most ? most : p * n;   // (an infinite product has no rest)
}

// 1 / sqrt(a) to the last bit but one: the hardware's value (1 ulp), corrected by what a r^2 is off from 1, in two parts.
__device__ __forceinline__ float inverse_root(float a) {
  const float r = __builtin_amdgcn_rsqf(a), t = a * r, rest = fmaf(a, r, -t);
  const float e = fmaf(-t, r, 1.f) - rest * r, better = fmaf(0.5f * r, e, r);
  return better == better ? better : r;   // (0, infinity, NaN, and numbers so small that a r is none)
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

template <typename T>
__global__ __launch_bounds__(kThreads) void norm_kernel(const T *x, const T *residual, const void *weight, bool wide, T *y,
                                                        unsigned char *q, float *scales, T *sum, long rows, int columns,
                                                        float eps) {
  __shared__ float lds[kThreads / 64];
  const long row = linear_block();
  if (row >= rows) return;
  const T *xr = x + row * columns;
  float squares = 0.f;
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
  const float n = inverse_root(block_sum(squares, lds) / columns + eps);
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
__global__ __launch_bounds__(kThreads) void norm_grad_rows(const T *h, const void *weight, bool wide, const T *gy, const T *gsum,
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
  if (threadIdx.x == 0) norms[row] = n;
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
__global__ __launch_bounds__(kThreads) void norm_grad_columns(const T *h, const T *gy, const float *norms, float *partial,
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

template <typename T>
__global__ __launch_bounds__(kThreads) void norm_grad_weight(const float *partial, void *gw, bool wide, int columns) {
  const int c = blockIdx.x * kThreads + threadIdx.x;
  if (c >= columns) return;
  float sum = 0.f;
  for (int s = 0; s < kSlices; ++s) sum += partial[static_cast<long>(s) * columns + c];
  if (wide) static_cast<float *>(gw)[c] = sum;
  else static_cast<T *>(gw)[c] = store_cast<T>(sum);
}

// One wavefront for four blocks of one row and 128 columns.
template <typename T>
__global__ __launch_bounds__(kThreads) void quantize_rows(const T *x, unsigned char *q, float *scales, long blocks, int columns) {
  const int per_row = (columns + kBlock - 1) / kBlock;
  const long block = static_cast<long>(linear_block()) * (kThreads / 16) + threadIdx.x / 16;
  if (block >= blocks) return;
  const long row = block / per_row;
  const int c = static_cast<int>(block % per_row) * kBlock + (threadIdx.x & 15) * 8;
  float v[8];
  load8(x + row * columns + c, columns - c, v);
  const float s = lanes_scale(v), inverse = 1.f / s;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] *= inverse;
  *reinterpret_cast<u32x2 *>(q + row * (static_cast<long>(per_row) * kBlock) + c) = to_e4m3(v);
  if ((threadIdx.x & 15) == 0) scales[block] = s;
}

// One workgroup for a block of 128 x 128: 16 rows at a time, twice.
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
  MV_FLOATS(dtype, norm_kernel<T><<<linear_grid(rows, kThreads), kThreads, 0, static_cast<hipStream_t>(stream)>>>(
      static_cast<const T *>(x), static_cast<const T *>(residual), weight, weight_dtype == MV_F32, static_cast<T *>(y),
      static_cast<unsigned char *>(q), static_cast<float *>(scales), static_cast<T *>(sum), rows, columns, eps))
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
  return 4 * (static_cast<size_t>(rows) + static_cast<size_t>(kSlices) * columns);
}

int mv_add_rms_norm_backward(const void *h, const void *weight, const void *grad_y, const void *grad_sum, void *grad_x,
                             void *grad_weight, int64_t rows, int columns, float eps, int dtype, int weight_dtype,
                             void *workspace, size_t workspace_bytes, void *stream) {
  if (const int status = norm_arguments(rows, columns, dtype, weight_dtype)) return status;
  MV_REQUIRE(weight && grad_weight && (rows == 0 || (h && grad_y && grad_x)), "a tensor is missing");
  MV_REQUIRE(workspace && workspace_bytes >= mv_add_rms_norm_backward_workspace_bytes(rows, columns), "the workspace is too small");
  float *const norms = static_cast<float *>(workspace), *const partial = norms + rows;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const bool wide = weight_dtype == MV_F32;
  MV_FLOATS(dtype, {
    if (rows > 0)
      norm_grad_rows<T><<<linear_grid(rows, kThreads), kThreads, 0, s>>>(
          static_cast<const T *>(h), weight, wide, static_cast<const T *>(grad_y), static_cast<const T *>(grad_sum),
          static_cast<T *>(grad_x), norms, rows, columns, eps);
    norm_grad_columns<T><<<dim3((columns + kThreads * 8 - 1) / (kThreads * 8), kSlices), kThreads, 0, s>>>(
        static_cast<const T *>(h), static_cast<const T *>(grad_y), norms, partial, rows, columns);
    norm_grad_weight<T><<<(columns + kThreads - 1) / kThreads, kThreads, 0, s>>>(partial, grad_weight, wide, columns);
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
      quantize_rows<T><<<linear_grid((rows * per_row * 16 + kThreads - 1) / kThreads, kThreads), kThreads, 0, s>>>(
          static_cast<const T *>(x), static_cast<unsigned char *>(q), static_cast<float *>(scales), rows * per_row, columns);
    else
      quantize_tiles<T><<<linear_grid((rows + kBlock - 1) / kBlock * per_row, kThreads), kThreads, 0, s>>>(
          static_cast<const T *>(x), static_cast<unsigned char *>(q), static_cast<float *>(scales), rows, columns);
  })
  return check_launch("quantize_blocks");
}

}  // extern "C"

// Sums of a split product: [splits, count] in 32 bits.
#pragma once
#include "rows.hpp"

namespace mv {

// The parts' sum, in a fixed order: `Slices` threads share the parts of a result.
template <typename T, int Slices>
__global__ __launch_bounds__(256) void join_parts(const float *part, const T *bias, T *y, long count, int outputs, int splits) {
  constexpr int kWide = 256 / Slices;
  __shared__ float sums[Slices][kWide];
  const int in = threadIdx.x % kWide, slice = threadIdx.x / kWide;
  const long at = static_cast<long>(linear_block()) * kWide + in;
  float sum = 0.f;
  if (at < count) {
#pragma unroll 4
    for (int s = slice; s < splits; s += Slices) sum += part[s * count + at];
  }
  if constexpr (Slices > 1) {
    sums[slice][in] = sum;
    __syncthreads();
    if (slice) return;
#pragma unroll
    for (int i = 1; i < Slices; ++i) sum += sums[i][in];
  }
  if (at >= count) return;
  if (bias) sum += load(bias + at % outputs);
  y[at] = store_cast<T>(sum);
}

// Four neighbouring results of a row per thread, for outputs in fours.
template <typename T>
__global__ __launch_bounds__(256) void join_fours(const float *part, const T *bias, T *y, long fours, unsigned row_fours, int splits) {
  const long at = static_cast<long>(linear_block()) * 256 + threadIdx.x;
  if (at >= fours) return;
  float sum[4] = {};
#pragma unroll 4
  for (int s = 0; s < splits; ++s) {
    const f32x4 v = reinterpret_cast<const Loose<f32x4, 4> *>(part + 4 * (s * fours + at))->v;
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[i] += v[i];
  }
  if (bias) {
    const T *const add = bias + 4 * (static_cast<unsigned long>(at) >> 32 ? at % row_fours : static_cast<unsigned>(at) % row_fours);
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[i] += load(add + i);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) y[4 * at + i] = store_cast<T>(sum[i]);
}

// Many parts are shared out over threads, results of fewer go in fours (four parts of 2000 x 1024: 7 us, one by one 8.5).
template <typename T> void launch_join(const float *part, const T *bias, T *y, long count, int outputs, int splits, hipStream_t s) {
  if (splits > 8) join_parts<T, 8><<<linear_grid((count + 31) / 32, 256), 256, 0, s>>>(part, bias, y, count, outputs, splits);
  else if (outputs % 4) join_parts<T, 1><<<linear_grid((count + 255) / 256, 256), 256, 0, s>>>(part, bias, y, count, outputs, splits);
  else join_fours<T><<<linear_grid((count / 4 + 255) / 256, 256), 256, 0, s>>>(part, bias, y, count / 4, outputs / 4, splits);
}

}  // namespace mv

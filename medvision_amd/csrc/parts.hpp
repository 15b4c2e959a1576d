// Sums of a split product: [splits, count] in 32 bits.
#pragma once
#include "common.hpp"

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

}  // namespace mv

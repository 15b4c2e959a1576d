// Group norm of small samples (group_norm_small.hip), for the entry points in group_norm.hip.
#pragma once
#include "common.hpp"

namespace mv {

// Values whose squares 32 bits do not hold (float16 has none) are scaled by this in front of their sums.
constexpr float kDown = 0x1p-100f;
constexpr double kUp = 0x1p100;
template <typename T> inline constexpr bool kFar = true;
template <> inline constexpr bool kFar<__half> = false;
__device__ __forceinline__ bool held(float v) { return v <= 3.402823466e38f; }   // (of a sum of squares; not NaN)

// A workgroup for a group of a sample, whose values stay in its registers.
struct Whole {
  int cells, channels, groups, group_channels, units, rows;   // units of V channels of a group, rows of cells at a time
};
struct WholePlan {
  Whole s;
  int threads, v, u;   // u: cells of a thread, 0: the sample is too large
};
WholePlan whole_plan(int batch, long cells, int channels, int groups, bool gradients);

// y and stats; gx (NULL: not wanted) and the channels' sums of gz and gz h, sums[sample][channel] (NULL: not wanted)
int group_norm_whole(const WholePlan &plan, const void *x, const void *weight, const void *bias, bool wide, void *y, float *stats, int batch, float eps,
                     int activation, float low, int dtype, hipStream_t stream);
int group_norm_whole_backward(const WholePlan &plan, const void *x, const void *gy, const float *stats, const void *weight, const void *bias, bool wide,
                              void *gx, float2 *sums, int batch, int activation, float low, int dtype, hipStream_t stream);

}  // namespace mv

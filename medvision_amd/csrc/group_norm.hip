// Group norm of cells in channels-last order with an activation, and its gradients.
//
//   h = (x - mean) r,  r = 1 / sqrt(var + eps)   over the cells of a sample and the channels of a group
//   z = h w + b,  y = a(z)
//   gz = gy a'(z)      db = sum gz      dw = sum gz h      (sums over samples and cells)
//   dx = r (w gz - mean(w gz) - h mean(w gz h))            (means as above)
//
// Sums over the cells are kept for each channel: a thread has eight neighbouring channels and a share of the cells, a
// workgroup joins its threads' shares, and a small kernel joins the workgroups' to those of a group.  Two kernels with a pass over
// memory each, then; bound by memory.
#include "rows.hpp"
#include "activation.hpp"

#include <algorithm>
#include <type_traits>

namespace mv {
namespace {

constexpr int kThreads = 256;

// What a launch works on.  A tile is up to 2048 channels (256 threads of eight), a chunk a share of a sample's cells.
struct Cells {
  long cells, each;   // of a sample, of a chunk
  int channels, groups, group_channels, tile_threads, tile_rows, chunks;
};

// Where a thread stands: channels from c on (`left` of them exist), cells first, first + step, ... below last.
struct Place {
  int c, left, row;
  long first, last, step, base;   // base: of the sample's first cell, in elements
  bool live;
};
__device__ __forceinline__ Place place_of(const Cells &s) {
  Place p;
  const int octet = threadIdx.x % s.tile_threads;
  p.row = threadIdx.x / s.tile_threads;
  p.c = (blockIdx.y * kThreads + octet) * 8;
  p.left = s.channels - p.c;
  p.first = blockIdx.x * s.each + p.row;
  p.last = min(s.cells, (blockIdx.x + 1) * s.each);
  p.step = s.tile_rows;
  p.base = static_cast<long>(blockIdx.z) * s.cells * s.channels;
  p.live = p.row < s.tile_rows && p.left > 0;
  return p;
}

// ---- forward ------------------------------------------------------------------------------------------------------
// Of a channel over a chunk's cells: its mean in two parts and the sum of squared differences from it.
struct Moments {
  float mean, rest, squares;
};
// partial[sample][chunk][channel].  A thread sums differences from the mean of its first cells, which keeps 32 bits enough
// where a channel's mean is far from zero; threads are joined in 64 bits.
template <typename T>
__global__ __launch_bounds__(kThreads) void group_sums(const T *x, Moments *partial, const Cells s) {
  __shared__ Moments shares[kThreads][8];
  const Place p = place_of(s);
  float middle[8] = {}, sum[8] = {}, squares[8] = {};
  const long mine = p.live && p.first < p.last ? (p.last - p.first + p.step - 1) / p.step : 0;
  if (mine) {
    constexpr int kFirst = 4;
    float v[kFirst][8];
    const T *const at = x + p.base + p.c;
    const int few = static_cast<int>(min(mine, static_cast<long>(kFirst)));
#pragma unroll
    for (int i = 0; i < kFirst; ++i) load8(at + (p.first + min(i, few - 1) * p.step) * s.channels, p.left, v[i]);
#pragma unroll
    for (int i = 0; i < 8; ++i) middle[i] = ((v[0][i] + v[1][i]) + (v[2][i] + v[3][i])) * 0.25f;
#pragma unroll
    for (int n = 0; n < kFirst; ++n)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = n < few ? v[n][i] - middle[i] : 0.f;
        sum[i] += d;
        squares[i] = fmaf(d, d, squares[i]);
      }
#pragma unroll 4
    for (long r = p.first + kFirst * p.step; r < p.last; r += p.step) {
      float u[8];
      load8(at + r * s.channels, p.left, u);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = u[i] - middle[i];
        sum[i] += d;
        squares[i] = fmaf(d, d, squares[i]);
      }
    }
    const float each = 1.f / static_cast<float>(mine);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float off = sum[i] * each;
      squares[i] = fmaxf(fmaf(-sum[i], off, squares[i]), 0.f) + (squares[i] - squares[i]);   // (NaN stays)
      sum[i] = off;
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) shares[threadIdx.x][i] = {middle[i], sum[i], squares[i]};
  __syncthreads();
  // a channel of the tile each: the rows' shares
  for (int k = threadIdx.x; k < s.tile_threads * 8; k += kThreads) {
    const int c = blockIdx.y * kThreads * 8 + k;
    if (c >= s.channels) continue;
    const long begin = blockIdx.x * s.each, all = min(s.cells, begin + s.each) - begin;
    double total = 0., rest = 0.;
    for (int r = 0; r < s.tile_rows; ++r) {
      const long n = r < all ? (all - r + s.tile_rows - 1) / s.tile_rows : 0;
      const Moments share = shares[r * s.tile_threads + k / 8][k % 8];
      const double mean = static_cast<double>(share.mean) + share.rest;
      if (n) total += mean * n, rest += share.squares + mean * mean * n;
    }
    const double mean = total / all;
    const float high = static_cast<float>(mean);
    partial[(static_cast<long>(blockIdx.z) * s.chunks + blockIdx.x) * s.channels + c] = {high, static_cast<float>(mean - high), static_cast<float>(rest - total * mean)};
  }
}

__device__ __forceinline__ double block_sum(double v, double *lds) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0.;
#pragma unroll
  for (int i = 0; i < kThreads / 64; ++i) v += lds[i];
  __syncthreads();
  return v;
}

// A group of a sample: stats[0], [1], [2] = mean, what rounding took from it, r.
__global__ __launch_bounds__(kThreads) void group_finish(const Moments *partial, float *stats, const Cells s, float eps, int batch) {
  __shared__ double lds[kThreads / 64];
  const unsigned id = linear_block();
  if (id >= static_cast<unsigned>(batch) * s.groups) return;
  const int b = id / s.groups, g = id % s.groups;
  const Moments *const from = partial + static_cast<long>(b) * s.chunks * s.channels + static_cast<long>(g) * s.group_channels;
  double total = 0., rest = 0.;
  for (long k = threadIdx.x; k < static_cast<long>(s.chunks) * s.group_channels; k += kThreads) {
    const long chunk = k / s.group_channels, c = k % s.group_channels;
    const double n = static_cast<double>(min(s.cells, (chunk + 1) * s.each) - chunk * s.each);
    const Moments share = from[chunk * s.channels + c];
    const double mean = static_cast<double>(share.mean) + share.rest;
    total += n * mean;
    rest += share.squares + n * mean * mean;
  }
  total = block_sum(total, lds);
  rest = block_sum(rest, lds);
  if (threadIdx.x) return;
  const double all = static_cast<double>(s.cells) * s.group_channels, mean = total / all;
  const double left = rest / all - mean * mean, var = left < 0. ? 0. : left;   // (NaN stays)
  const long at = id, every = static_cast<long>(batch) * s.groups;
  stats[at] = static_cast<float>(mean);
  stats[every + at] = static_cast<float>(mean - static_cast<float>(mean));
  stats[2 * every + at] = static_cast<float>(1. / sqrt(var + eps));
}

template <typename T> __device__ __forceinline__ float vector_at(const void *w, bool wide, int c, float absent) {
  return !w ? absent : wide ? static_cast<const float *>(w)[c] : load(static_cast<const T *>(w) + c);
}

// What the channels of a thread need
struct Channels {
  float mean[8], rest[8], r[8], w[8], b[8];
};
template <typename T>
__device__ __forceinline__ void load_channels(Channels &t, const Place &p, const float *stats, const void *weight, const void *bias, bool wide,
                                              const Cells &s) {
  const long every = static_cast<long>(gridDim.z) * s.groups, first = static_cast<long>(blockIdx.z) * s.groups;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int c = min(p.c + i, s.channels - 1);
    const long at = first + c / s.group_channels;
    t.mean[i] = stats[at], t.rest[i] = stats[every + at], t.r[i] = stats[2 * every + at];
    t.w[i] = vector_at<T>(weight, wide, c, 1.f), t.b[i] = vector_at<T>(bias, wide, c, 0.f);
  }
}

template <typename T, int Kind>
__global__ __launch_bounds__(kThreads) void group_apply(const T *x, const float *stats, const void *weight, const void *bias, bool wide, T *y,
                                                        const Cells s, float low) {
  const Place p = place_of(s);
  if (!p.live) return;
  Channels t;
  load_channels<T>(t, p, stats, weight, bias, wide, s);
#pragma unroll 4
  for (long r = p.first; r < p.last; r += p.step) {
    const long at = p.base + r * s.channels + p.c;
    float v[8];
    load8(x + at, p.left, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = Activation<Kind>::value(fmaf(((v[i] - t.mean[i]) - t.rest[i]) * t.r[i], t.w[i], t.b[i]), low);
    store8(y + at, p.left, v);
  }
}

// ---- gradients ------------------------------------------------------------------------------------------------------
// Sums of gz and gz h of each channel over a chunk's cells
template <typename T, int Kind>
__global__ __launch_bounds__(kThreads) void group_grad_sums(const T *x, const T *gy, const float *stats, const void *weight, const void *bias,
                                                            bool wide, float2 *partial, const Cells s, float low) {
  __shared__ float2 shares[kThreads][8 + 1];
  const Place p = place_of(s);
  float sum[8] = {}, dot[8] = {};
  if (p.live) {
    Channels t;
    load_channels<T>(t, p, stats, weight, bias, wide, s);
#pragma unroll 4
    for (long r = p.first; r < p.last; r += p.step) {
      const long at = p.base + r * s.channels + p.c;
      float v[8], g[8];
      load8(x + at, p.left, v);
      load8(gy + at, p.left, g);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float h = ((v[i] - t.mean[i]) - t.rest[i]) * t.r[i], gz = g[i] * Activation<Kind>::slope(fmaf(h, t.w[i], t.b[i]), low);
        sum[i] += gz;
        dot[i] = fmaf(gz, h, dot[i]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) shares[threadIdx.x][i] = {sum[i], dot[i]};
  __syncthreads();
  for (int k = threadIdx.x; k < s.tile_threads * 8; k += kThreads) {
    const int c = blockIdx.y * kThreads * 8 + k;
    if (c >= s.channels) continue;
    float2 all = {0.f, 0.f};
    for (int r = 0; r < s.tile_rows; ++r) {
      const float2 share = shares[r * s.tile_threads + k / 8][k % 8];
      all.x += share.x, all.y += share.y;
    }
    partial[(static_cast<long>(blockIdx.z) * s.chunks + blockIdx.x) * s.channels + c] = all;
  }
}

// A group of a sample: means[0], [1] = mean(w gz), mean(w gz h); the channels' sums over all chunks take the first one's place.
template <typename T>
__global__ __launch_bounds__(kThreads) void group_grad_finish(float2 *partial, float *means, const void *weight, bool wide, const Cells s, int batch) {
  __shared__ double lds[kThreads / 64];
  const unsigned id = linear_block();
  if (id >= static_cast<unsigned>(batch) * s.groups) return;
  const int b = id / s.groups, g = id % s.groups;
  float2 *const from = partial + static_cast<long>(b) * s.chunks * s.channels + static_cast<long>(g) * s.group_channels;
  double sum = 0., dot = 0.;
  for (int c = 0; c < s.group_channels; ++c) {
    double one = 0., two = 0.;
    for (long chunk = threadIdx.x; chunk < s.chunks; chunk += kThreads) {
      const float2 share = from[chunk * s.channels + c];
      one += share.x, two += share.y;
    }
    one = block_sum(one, lds);
    two = block_sum(two, lds);
    if (threadIdx.x == 0) from[c] = {static_cast<float>(one), static_cast<float>(two)};
    const double w = vector_at<T>(weight, wide, g * s.group_channels + c, 1.f);
    sum += w * one, dot += w * two;
  }
  if (threadIdx.x) return;
  const double all = static_cast<double>(s.cells) * s.group_channels;
  means[id] = static_cast<float>(sum / all);
  means[static_cast<long>(batch) * s.groups + id] = static_cast<float>(dot / all);
}

template <typename T, int Kind>
__global__ __launch_bounds__(kThreads) void group_grad_apply(const T *x, const T *gy, const float *stats, const float *means, const void *weight,
                                                             const void *bias, bool wide, T *gx, const Cells s, float low) {
  const Place p = place_of(s);
  if (!p.live) return;
  Channels t;
  load_channels<T>(t, p, stats, weight, bias, wide, s);
  float one[8], two[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const long at = static_cast<long>(blockIdx.z) * s.groups + min(p.c + i, s.channels - 1) / s.group_channels;
    one[i] = means[at], two[i] = means[static_cast<long>(gridDim.z) * s.groups + at];
  }
#pragma unroll 2
  for (long r = p.first; r < p.last; r += p.step) {
    const long at = p.base + r * s.channels + p.c;
    float v[8], g[8];
    load8(x + at, p.left, v);
    load8(gy + at, p.left, g);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float h = ((v[i] - t.mean[i]) - t.rest[i]) * t.r[i], gz = g[i] * Activation<Kind>::slope(fmaf(h, t.w[i], t.b[i]), low);
      v[i] = t.r[i] * (fmaf(gz, t.w[i], -one[i]) - h * two[i]);
    }
    store8(gx + at, p.left, v);
  }
}

// Sums of the channels over the samples, in their order
template <typename T>
__global__ __launch_bounds__(kThreads) void group_grad_vectors(const float2 *partial, void *gw, void *gb, bool wide, const Cells s, int batch) {
  const int c = blockIdx.x * kThreads + threadIdx.x;
  if (c >= s.channels) return;
  double sum = 0., dot = 0.;
  for (int b = 0; b < batch; ++b) {
    const float2 share = partial[static_cast<long>(b) * s.chunks * s.channels + c];
    sum += share.x, dot += share.y;
  }
  auto put = [&](void *to, double v) {
    if (!to) return;
    if (wide) static_cast<float *>(to)[c] = static_cast<float>(v);
    else static_cast<T *>(to)[c] = store_cast<T>(static_cast<float>(v));
  };
  put(gb, sum);
  put(gw, dot);
}

// ---- launches -------------------------------------------------------------------------------------------------------
Cells cells_of(int batch, long cells, int channels, int groups) {
  Cells s{};
  s.cells = cells, s.channels = channels, s.groups = groups, s.group_channels = channels / groups;
  const int octets = (channels + 7) / 8, tiles = (octets + kThreads - 1) / kThreads;
  s.tile_threads = std::min(octets, kThreads), s.tile_rows = kThreads / s.tile_threads;
  // about eight workgroups per compute unit, of eight cells a thread at least
  const long most = std::max(1L, 2048L / std::max(1L, static_cast<long>(batch) * tiles)), rows = 8L * s.tile_rows;
  s.each = std::max(rows, (cells + most - 1) / most);
  s.each = (s.each + s.tile_rows - 1) / s.tile_rows * s.tile_rows;
  s.chunks = static_cast<int>(std::max(1L, (cells + s.each - 1) / s.each));
  return s;
}
int tiles_of(const Cells &s) { return ((s.channels + 7) / 8 + kThreads - 1) / kThreads; }

int arguments(int batch, long cells, int channels, int groups, int activation, int dtype, int weight_dtype) {
  MV_REQUIRE(dtype == MV_F32 || dtype == MV_F16 || dtype == MV_BF16, "dtype %d is not float32, float16 or bfloat16", dtype);
  MV_REQUIRE(weight_dtype == dtype || weight_dtype == MV_F32, "weight and bias have dtype %d, expected %d or float32", weight_dtype, dtype);
  MV_REQUIRE(batch >= 0 && batch < 65536 && cells >= 0 && cells < (1L << 40) && channels > 0 && channels <= (1 << 24), "wrong sizes: a batch of %d, %ld cells of %d channels", batch, cells, channels);
  MV_REQUIRE(groups > 0 && channels % groups == 0, "%d channels in %d groups", channels, groups);
  MV_REQUIRE(static_cast<long>(batch) * groups < (1L << 31), "too many groups: %d in a batch of %d", groups, batch);
  MV_REQUIRE(activation >= MV_NO_ACTIVATION && activation <= MV_GELU, "unknown activation %d", activation);
  return MV_OK;
}

template <typename Share> size_t partial_bytes(int batch, const Cells &s) { return sizeof(Share) * batch * s.chunks * static_cast<size_t>(s.channels); }

}  // namespace
}  // namespace mv

using namespace mv;

extern "C" {

size_t mv_group_norm_workspace_bytes(int batch, int64_t cells, int channels, int groups) {
  if (batch <= 0 || cells <= 0 || channels <= 0 || groups <= 0 || channels % groups) return 0;
  return partial_bytes<Moments>(batch, cells_of(batch, cells, channels, groups));
}

int mv_group_norm(const void *x, const void *weight, const void *bias, void *y, void *stats, int batch, int64_t cells, int channels,
                  int groups, float eps, int activation, float low, int dtype, int weight_dtype, void *workspace, size_t workspace_bytes,
                  void *stream) {
  if (const int status = arguments(batch, cells, channels, groups, activation, dtype, weight_dtype)) return status;
  if (batch == 0 || cells == 0) return MV_OK;
  MV_REQUIRE(x && y && stats, "a tensor is missing");
  MV_REQUIRE(workspace && workspace_bytes >= mv_group_norm_workspace_bytes(batch, cells, channels, groups), "the workspace is too small");
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const Cells s = cells_of(batch, cells, channels, groups);
  const dim3 grid(s.chunks, tiles_of(s), batch);
  const bool wide = weight_dtype == MV_F32;
  auto *const partial = static_cast<Moments *>(workspace);
  auto *const stat = static_cast<float *>(stats);
  MV_FLOATS(dtype, {
    const T *const xt = static_cast<const T *>(x);
    group_sums<T><<<grid, kThreads, 0, st>>>(xt, partial, s);
    group_finish<<<linear_grid(static_cast<long>(batch) * groups, kThreads), kThreads, 0, st>>>(partial, stat, s, eps, batch);
    for_activation(activation, [&](auto kind) {
      group_apply<T, kind><<<grid, kThreads, 0, st>>>(xt, stat, weight, bias, wide, static_cast<T *>(y), s, low);
    });
  })
  return check_launch("group_norm");
}

size_t mv_group_norm_backward_workspace_bytes(int batch, int64_t cells, int channels, int groups) {
  if (batch <= 0 || cells <= 0 || channels <= 0 || groups <= 0 || channels % groups) return 0;
  return partial_bytes<float2>(batch, cells_of(batch, cells, channels, groups)) + sizeof(float) * 2 * batch * groups;
}

int mv_group_norm_backward(const void *x, const void *weight, const void *bias, const void *stats, const void *grad_y, void *grad_x,
                           void *grad_weight, void *grad_bias, int batch, int64_t cells, int channels, int groups, int activation, float low,
                           int dtype, int weight_dtype, void *workspace, size_t workspace_bytes, void *stream) {
  if (const int status = arguments(batch, cells, channels, groups, activation, dtype, weight_dtype)) return status;
  const bool empty = batch == 0 || cells == 0;
  if ((empty || !grad_x) && !grad_weight && !grad_bias) return MV_OK;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const Cells s = cells_of(batch, cells, channels, groups);
  const bool wide = weight_dtype == MV_F32;
  MV_REQUIRE(empty || (x && stats && grad_y), "a tensor is missing");
  MV_REQUIRE(empty || (workspace && workspace_bytes >= mv_group_norm_backward_workspace_bytes(batch, cells, channels, groups)), "the workspace is too small");
  const dim3 grid(s.chunks, tiles_of(s), batch);
  auto *const partial = static_cast<float2 *>(workspace);
  auto *const means = reinterpret_cast<float *>(static_cast<char *>(workspace) + (empty ? 0 : partial_bytes<float2>(batch, s)));
  auto *const stat = static_cast<const float *>(stats);
  MV_FLOATS(dtype, {
    const T *const xt = static_cast<const T *>(x), *const gy = static_cast<const T *>(grad_y);
    if (!empty) {
      for_activation(activation, [&](auto kind) {
        group_grad_sums<T, kind><<<grid, kThreads, 0, st>>>(xt, gy, stat, weight, bias, wide, partial, s, low);
      });
      group_grad_finish<T><<<linear_grid(static_cast<long>(batch) * groups, kThreads), kThreads, 0, st>>>(partial, means, weight, wide, s, batch);
      if (grad_x)
        for_activation(activation, [&](auto kind) {
          group_grad_apply<T, kind><<<grid, kThreads, 0, st>>>(xt, gy, stat, means, weight, bias, wide, static_cast<T *>(grad_x), s, low);
        });
    }
    if (grad_weight || grad_bias)
      group_grad_vectors<T><<<(channels + kThreads - 1) / kThreads, kThreads, 0, st>>>(partial, grad_weight, grad_bias, wide, s, empty ? 0 : batch);
  })
  return check_launch("group_norm backward");
}

}  // extern "C"

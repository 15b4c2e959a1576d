// Group norm with an activation, and its gradients, of small samples (the mathematics stands in group_norm.hip): a workgroup
// for a group of a sample, whose values stay in registers.  One launch, one pass over memory; bound by the launch and by the way
// from one sum over the workgroup to the next.
//
// A thread has V neighbouring channels (V divides those of the group, so that all its values are of one group) of up to U
// cells: 64 / V and no more than 16; for gradients 32 / V.
#include "activation.hpp"
#include "group_norm.hpp"
#include "rows.hpp"

#include <algorithm>
#include <type_traits>

namespace mv {
namespace {

template <typename T, int V> struct Few {
  typedef unsigned short u16 __attribute__((ext_vector_type(V)));
  typedef unsigned u32 __attribute__((ext_vector_type(V)));
  std::conditional_t<sizeof(T) == 4, u32, u16> bits;
  __device__ __forceinline__ void load(const T *p) { bits = reinterpret_cast<const Loose<decltype(bits), sizeof(T)> *>(p)->v; }
  __device__ __forceinline__ float value(int i) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(bits[i]);
    else return Bits<T>::up(bits[i]);
  }
  __device__ __forceinline__ void put(int i, float v) {
    if constexpr (sizeof(T) == 4) bits[i] = __float_as_uint(v);
    else bits[i] = __builtin_bit_cast(unsigned short, store_cast<T>(v));
  }
  __device__ __forceinline__ void store(T *p) const { reinterpret_cast<Loose<decltype(bits), sizeof(T)> *>(p)->v = bits; }
};

// The sum over a workgroup of up to 1024 threads, the same for every thread
template <typename S> __device__ __forceinline__ S group_sum(S v) {
  __shared__ S lds[16];
#pragma unroll
  for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
  if (blockDim.x == 64) return v;
  __syncthreads();   // (the sum before this one has been read)
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0;
  for (int i = 0; i < static_cast<int>(blockDim.x >> 6); ++i) v += lds[i];
  return v;
}

// Where a thread of group g of sample b stands
struct Spot {
  int b, g, c, row;
  long base;   // of its first channel in the sample's first cell
  bool live;
};
template <int V> __device__ __forceinline__ Spot spot_of(const Whole &s, unsigned id) {
  Spot p;
  p.b = id / s.groups, p.g = id % s.groups;
  p.row = threadIdx.x / s.units;
  p.c = p.g * s.group_channels + static_cast<int>(threadIdx.x - p.row * s.units) * V;
  p.base = static_cast<long>(p.b) * s.cells * s.channels + p.c;
  p.live = p.row < s.rows;
  return p;
}
template <typename T, int V> __device__ __forceinline__ void few_at(float (&to)[V], const void *w, bool wide, int c, float absent) {
#pragma unroll
  for (int i = 0; i < V; ++i) to[i] = absent;
  if (!w) return;
  if (wide) {
    Few<float, V> raw;
    raw.load(static_cast<const float *>(w) + c);
#pragma unroll
    for (int i = 0; i < V; ++i) to[i] = raw.value(i);
  } else {
    Few<T, V> raw;
    raw.load(static_cast<const T *>(w) + c);
#pragma unroll
    for (int i = 0; i < V; ++i) to[i] = raw.value(i);
  }
}

template <typename T, int V, int U, int Kind>
__global__ __launch_bounds__(1024) void group_whole(const T *x, const void *weight, const void *bias, bool wide, T *y, float *stats, const Whole s,
                                                    float eps, float low, unsigned count) {
  if (linear_block() >= count) return;
  const unsigned id = xcd_contiguous(linear_block(), count);   // (neighbouring groups share cache lines)
  const Spot p = spot_of<V>(s, id);
  Few<T, V> raw[U];
#pragma unroll
  for (int n = 0; n < U; ++n) raw[n].load(x + p.base + static_cast<long>(min(p.row + n * s.rows, s.cells - 1)) * s.channels);
  float w[V], b[V];
  few_at<T, V>(w, weight, wide, p.c, 1.f);
  few_at<T, V>(b, bias, wide, p.c, 0.f);
  const int mine = p.live ? (s.cells - p.row + s.rows - 1) / s.rows : 0;   // (0 or less: none)
  const double all = static_cast<double>(s.cells) * s.group_channels;
  double mean, var;
  auto moments = [&](auto scaled) {   // of the values, or of them times kDown
    float sum = 0.f;
#pragma unroll
    for (int n = 0; n < U; ++n)
      if (n < mine) {
#pragma unroll
        for (int i = 0; i < V; ++i) sum += scaled ? raw[n].value(i) * kDown : raw[n].value(i);
      }
    const float middle = static_cast<float>(group_sum(sum) / all);   // about the mean: differences from it are small
    float off = 0.f, squares = 0.f;
#pragma unroll
    for (int n = 0; n < U; ++n)
      if (n < mine) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float d = scaled ? fmaf(raw[n].value(i), kDown, -middle) : raw[n].value(i) - middle;
          off += d;
          squares = fmaf(d, d, squares);
        }
      }
    const double total = group_sum(static_cast<double>(off)), rest = group_sum(static_cast<double>(squares));
    const double shift = total / all, left = rest / all - shift * shift;
    mean = middle + shift, var = left < 0. ? 0. : left;   // (NaN stays)
  };
  moments(std::false_type());
  if constexpr (kFar<T>) {
    if (!(var < 1e300)) {   // squares that 32 bits do not hold (the same for every thread)
      moments(std::true_type());
      mean *= kUp, var *= kUp * kUp;
    }
  }
  const float high = static_cast<float>(mean), small = static_cast<float>(mean - high), r = static_cast<float>(1. / sqrt(var + eps));
  if (threadIdx.x == 0) stats[id] = high, stats[count + id] = small, stats[2L * count + id] = r;
#pragma unroll
  for (int n = 0; n < U; ++n)
    if (n < mine) {
#pragma unroll
      for (int i = 0; i < V; ++i) raw[n].put(i, Activation<Kind>::value(fmaf(((raw[n].value(i) - high) - small) * r, w[i], b[i]), low));
      raw[n].store(y + p.base + static_cast<long>(p.row + n * s.rows) * s.channels);
    }
}

// Every step-th of the rows from the first, in 64 bits
__device__ __forceinline__ float2 join_rows(const float2 *column, int first, int step, int lines, int channels) {
  double t = 0., u = 0.;
#pragma unroll 4
  for (int k = first; k < lines; k += step) t += column[k * channels].x, u += column[k * channels].y;
  return {static_cast<float>(t), static_cast<float>(u)};
}

// The gradients of a group of a sample: gx, and the sums of its channels, sums[sample][channel].
template <typename T, int V, int U, int Kind>
__global__ __launch_bounds__(1024) void group_grad_whole(const T *x, const T *gy, const float *stats, const void *weight, const void *bias, bool wide, T *gx,
                                                         float2 *sums, const Whole s, float low, unsigned count) {
  extern __shared__ float2 rows[];   // of a wavefront's rows, or of every row: the channels' sums
  if (linear_block() >= count) return;
  const unsigned id = xcd_contiguous(linear_block(), count);
  const Spot p = spot_of<V>(s, id);
  Few<T, V> raw[U], graw[U];
#pragma unroll
  for (int n = 0; n < U; ++n) {
    const long at = p.base + static_cast<long>(min(p.row + n * s.rows, s.cells - 1)) * s.channels;
    raw[n].load(x + at);
    graw[n].load(gy + at);
  }
  float w[V], b[V], one[V] = {}, two[V] = {};
  few_at<T, V>(w, weight, wide, p.c, 1.f);
  few_at<T, V>(b, bias, wide, p.c, 0.f);
  const float high = stats[id], small = stats[count + id], r = stats[2L * count + id];
  const int mine = p.live ? (s.cells - p.row + s.rows - 1) / s.rows : 0;
  float sum = 0.f, dot = 0.f;
#pragma unroll
  for (int n = 0; n < U; ++n)
    if (n < mine) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float h = ((raw[n].value(i) - high) - small) * r, gz = graw[n].value(i) * Activation<Kind>::slope(fmaf(h, w[i], b[i]), low);
        one[i] += gz;
        two[i] = fmaf(gz, h, two[i]);
      }
    }
#pragma unroll
  for (int i = 0; i < V; ++i) sum = fmaf(w[i], one[i], sum), dot = fmaf(w[i], two[i], dot);
  if (gx) {
    const double all = static_cast<double>(s.cells) * s.group_channels;
    const float first = static_cast<float>(group_sum(static_cast<double>(sum)) / all), second = static_cast<float>(group_sum(static_cast<double>(dot)) / all);
#pragma unroll
    for (int n = 0; n < U; ++n)
      if (n < mine) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float h = ((raw[n].value(i) - high) - small) * r, gz = graw[n].value(i) * Activation<Kind>::slope(fmaf(h, w[i], b[i]), low);
          raw[n].put(i, r * (fmaf(gz, w[i], -first) - h * second));
        }
        raw[n].store(gx + p.base + static_cast<long>(p.row + n * s.rows) * s.channels);
      }
  }
  if (!sums) return;
  // Rows of a wavefront first, where its lanes have the units side by side as often as they go into it
  int lines = s.rows, line = p.row;
  const int unit = threadIdx.x - p.row * s.units;
  bool puts = p.live;
  if (s.units < 64 && (s.units & (s.units - 1)) == 0) {
    for (int d = s.units; d < 64; d *= 2) {
#pragma unroll
      for (int i = 0; i < V; ++i) one[i] += __shfl_xor(one[i], d), two[i] += __shfl_xor(two[i], d);
    }
    lines = blockDim.x >> 6, line = threadIdx.x >> 6, puts = static_cast<int>(threadIdx.x & 63) < s.units;
  }
  if (puts) {
#pragma unroll
    for (int i = 0; i < V; ++i) rows[line * s.group_channels + unit % s.units * V + i] = {one[i], two[i]};
  }
  __syncthreads();
  // Then sixteen threads to a channel (each leaves its sum in the first row that it reads, which no other reads), and one over their sums:
  // 3 x 1955 x 60 in 6 groups 15.4 us, with one thread to a channel 18
  const int strides = min(16, static_cast<int>(blockDim.x) / s.group_channels);
  if (strides > 1 && lines > strides) {
    const int c = threadIdx.x % s.group_channels, first = threadIdx.x / s.group_channels;
    if (first < strides) rows[first * s.group_channels + c] = join_rows(rows + c, first, strides, lines, s.group_channels);
    __syncthreads();
    lines = strides;
  }
  for (int c = threadIdx.x; c < s.group_channels; c += blockDim.x)
    sums[static_cast<long>(p.b) * s.channels + p.g * s.group_channels + c] = join_rows(rows + c, 0, 1, lines, s.group_channels);
}

constexpr int forward_cells(int v) { return 64 / v > 16 ? 16 : 64 / v; }
constexpr int grad_cells(int v) { return v <= 2 ? 16 : forward_cells(v) / 2; }
bool folds(const Whole &s) { return s.units < 64 && (s.units & (s.units - 1)) == 0; }

// Calls f with V and U of a plan, as constants
template <bool Gradients, typename F> void for_plan(const WholePlan &p, const F &f) {
  using std::integral_constant;
  const auto with = [&](auto v) {
    constexpr int kMost = Gradients ? grad_cells(v) : forward_cells(v);
    if (p.u == 2) f(v, integral_constant<int, 2>());
    else f(v, integral_constant<int, kMost>());
  };
  switch (p.v) {
    case 8: with(integral_constant<int, 8>()); break;
    case 4: with(integral_constant<int, 4>()); break;
    case 2: with(integral_constant<int, 2>()); break;
    default: with(integral_constant<int, 1>());
  }
}

}  // namespace

// V is the largest power of two up to 8 that divides a group's channels.  A workgroup reads as many cache lines as there are cells, by itself:
// 8 x 5000 cells of 20 channels in groups of 4 8.9 us (12.3 in the three kernels of large samples), 8000 of 32 in groups of 8 16.4
// (13.4).  Gradients read two tensors, and keep the chip's other workgroups waiting where there are many: 4 x 2000 of 64 in groups of 4
// 11 us (16), 1 x 4000 of 256 in groups of 8 18 (15), 64 x 343 of 256 29 (26).  (Batches of 65536 and more, which are
// taken for the sake of this form, have it for gradients wherever it holds them.)
WholePlan whole_plan(int batch, long cells, int channels, int groups, bool gradients) {
  WholePlan p{};
  if (cells > (gradients ? 3000 : 5000) || (gradients && batch * cells * channels > (4L << 20) && batch < 65536)) return p;
  const int each = channels / groups;
  p.v = each % 8 == 0 ? 8 : each % 4 == 0 ? 4 : each % 2 == 0 ? 2 : 1;
  p.s = {0, channels, groups, each, each / p.v, 0};
  const int most = gradients ? grad_cells(p.v) : forward_cells(p.v), most_threads = gradients && !folds(p.s) && p.v == 8 ? 512 : 1024;   // (sums of each row in LDS: 32 KB)
  if (p.s.units > most_threads || cells > static_cast<long>(most_threads / p.s.units) * most) return p;
  p.threads = 64;   // two cells a thread while there are threads
  while (p.threads < most_threads && cells > 2L * (p.threads / p.s.units)) p.threads *= 2;
  p.s.cells = static_cast<int>(cells), p.s.rows = p.threads / p.s.units;
  p.u = cells <= 2L * p.s.rows ? 2 : most;
  return p;
}

int group_norm_whole(const WholePlan &plan, const void *x, const void *weight, const void *bias, bool wide, void *y, float *stats, int batch, float eps,
                     int activation, float low, int dtype, hipStream_t stream) {
  const unsigned count = static_cast<unsigned>(batch) * plan.s.groups;
  MV_FLOATS(dtype, {
    for_activation(activation, [&](auto kind) {
      for_plan<false>(plan, [&](auto v, auto u) {
        group_whole<T, v, u, kind><<<linear_grid(count, plan.threads), plan.threads, 0, stream>>>(static_cast<const T *>(x), weight, bias, wide,
                                                                                                  static_cast<T *>(y), stats, plan.s, eps, low, count);
      });
    });
  })
  return check_launch("group_norm");
}

int group_norm_whole_backward(const WholePlan &plan, const void *x, const void *gy, const float *stats, const void *weight, const void *bias, bool wide,
                              void *gx, float2 *sums, int batch, int activation, float low, int dtype, hipStream_t stream) {
  const unsigned count = static_cast<unsigned>(batch) * plan.s.groups;
  const size_t lds = sizeof(float2) * (folds(plan.s) ? plan.threads / 64 : plan.s.rows) * plan.s.group_channels;
  MV_FLOATS(dtype, {
    for_activation(activation, [&](auto kind) {
      for_plan<true>(plan, [&](auto v, auto u) {
        group_grad_whole<T, v, u, kind><<<linear_grid(count, plan.threads), plan.threads, lds, stream>>>(
            static_cast<const T *>(x), static_cast<const T *>(gy), stats, weight, bias, wide, static_cast<T *>(gx), sums, plan.s, low, count);
      });
    });
  })
  return check_launch("group_norm backward");
}

}  // namespace mv

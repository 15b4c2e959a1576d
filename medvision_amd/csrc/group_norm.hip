// Group norm of cells in channels-last order with an activation, and its gradients.
//
//   h = (x - mean) r,  r = 1 / sqrt(var + eps)   over the cells of a sample and the channels of a group
//   z = h w + b,  y = a(z)
//   gz = gy a'(z)      db = sum gz      dw = sum gz h      (sums over samples and cells)
//   dx = r (w gz - mean(w gz) - h mean(w gz h))            (means as above)
//
// Sums over the cells are kept for each channel: a thread has eight neighbouring channels and a share of the cells, a
// workgroup joins its threads' shares, and a small kernel joins the workgroups' to those of a group.  Two kernels with a pass over
// memory each, then; bound by memory: 2 x 128^3 cells of 32 channels in float16 (268 MB a pass) 60 us the sums, 5 the join, 95 the second
// pass; gradients 109 and 159 us, 7 the join (4.5 - 5.6 TB/s, about a copy's 4.9).  2 x 27648 cells of 256 channels in bf16, which caches
// hold: 9, 4, and 12 us with SiLU; the exact GELU's instructions make it 16.
#include "activation.hpp"
#include "group_norm.hpp"
#include "rows.hpp"

#include <algorithm>
#include <type_traits>

namespace mv {
namespace {

constexpr int kThreads = 256;

// What a launch works on.  A tile is up to 2048 channels (256 threads of eight), a chunk a share of a sample's cells.
struct Cells {
  long cells, each;   // of a sample, of a chunk
  int channels, groups, group_channels, tile_threads, tile_rows, chunks;
  int batch, first;   // all samples, the launch's first one
};
__device__ __forceinline__ long sample_of(const Cells &s) { return static_cast<long>(s.first) + blockIdx.z; }

// The first channel of a piece of eight.  The last piece starts earlier than its place where it would not be whole: the channels
// that it has in common with the one before are worked out twice, with the same results.
__device__ __forceinline__ int first_channel(const Cells &s, int octet) { return max(0, min(octet * 8, s.channels - 8)); }

// Cells of a chunk, and those of them that a row of a tile takes.  (In 32 bits, and divided once for a workgroup: divisions in 64 bits by
// each thread and row took the sums of 2 x 27648 cells of 256 channels from 9.2 to 11.4 us.)
__device__ __forceinline__ int cells_in(const Cells &s, unsigned chunk) { return static_cast<int>(min(s.each, s.cells - chunk * s.each)); }
struct Rows {
  int each, more;
  __device__ __forceinline__ Rows(const Cells &s, int cells) : each(cells / s.tile_rows), more(cells % s.tile_rows) {}
  __device__ __forceinline__ int of(int row) const { return each + (row < more ? 1 : 0); }
};

// Where a thread stands: channels from c on (`left` of them exist), `cells` cells that are `stride` elements apart, the first one
// `at` elements from the start.
struct Place {
  int c, left, cells;
  long stride, at;
};
__device__ __forceinline__ Place place_of(const Cells &s, unsigned chunk) {
  Place p;
  const int octet = threadIdx.x % s.tile_threads, row = threadIdx.x / s.tile_threads;
  const int piece = blockIdx.y * kThreads + octet;
  p.c = first_channel(s, piece);
  p.left = s.channels - piece * 8 > 0 ? s.channels - p.c : 0;
  p.cells = row < s.tile_rows && p.left > 0 ? Rows(s, cells_in(s, chunk)).of(row) : 0;
  p.stride = static_cast<long>(s.tile_rows) * s.channels;
  p.at = (sample_of(s) * s.cells + chunk * s.each + row) * s.channels + p.c;
  return p;
}

// How a kernel's pieces of eight channels are read and written: one element after the other (fewer than eight channels), whole, or
// whole with results that go past the caches.
enum Form { kParts, kWhole, kWholePast };

// Eight channels of a cell: as they are in memory where all of them exist, so that several cells' loads are on their way before the
// first is used.
template <typename T, int F> struct Eight {
  Raw<T> raw;
  __device__ __forceinline__ void load(const T *p, int) { raw.load(p); }
  __device__ __forceinline__ void values(float (&v)[8]) const { raw.values(v); }
};
template <typename T> struct Eight<T, kParts> {
  float v[8];
  __device__ __forceinline__ void load(const T *p, int left) { load8(p, left, v); }
  __device__ __forceinline__ void values(float (&out)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = v[i];
  }
};
// Results of more than what caches hold go past them (2 x 128^3 cells of 32 channels in float16: 160 instead of 177 us, gradients 283
// instead of 294).
template <typename T, int F> __device__ __forceinline__ void put_eight(T *p, int left, const float (&v)[8]) {
  if constexpr (F == kWholePast) {
    Raw<T> raw;
    raw.set(v);
#pragma unroll
    for (unsigned i = 0; i < sizeof(T) / 2; ++i) __builtin_nontemporal_store(raw.bits[i], &reinterpret_cast<Loose<u32x4, sizeof(T)> *>(p)[i].v);
  } else {
    store8(p, F == kWhole ? 8 : left, v);
  }
}
// Pieces of kAtOnce cells, the last one again where there are fewer left.
constexpr int kAtOnce = 4;
template <typename T, int F>
__device__ __forceinline__ void load_cells(Eight<T, F> (&to)[kAtOnce], const T *at, int cells, const Place &p) {
#pragma unroll
  for (int n = 0; n < kAtOnce; ++n) to[n].load(at + min(n, cells - 1) * p.stride, p.left);
}

// What the rows of a tile have of each of its channels, joined by teams of threads and then over the teams, in a fixed order:
// add(first row, step, piece, channel of it, sum), put(channel, sum).
template <typename Sum, typename Add, typename Put> __device__ __forceinline__ void join_rows(const Cells &s, const Add &add, const Put &put) {
  __shared__ Sum sums[kThreads];
  const int wide = min(s.tile_threads * 8, kThreads), team = threadIdx.x / wide, teams = kThreads / wide;
  for (int first = 0; first < s.tile_threads * 8; first += wide) {
    const int k = first + threadIdx.x % wide, c = blockIdx.y * kThreads * 8 + k;
    const bool mine = team < teams && k < s.tile_threads * 8 && c < s.channels;
    Sum all = {0, 0};
    if (mine) add(team, teams, k / 8, c - first_channel(s, c / 8), all);
    if (teams > 1) {
      sums[threadIdx.x] = all;
      __syncthreads();
      if (mine && team == 0)
        for (int t = 1; t < teams; ++t) all.x += sums[t * wide + k].x, all.y += sums[t * wide + k].y;
    }
    if (mine && team == 0) put(c, all);
  }
}

// ---- forward ------------------------------------------------------------------------------------------------------
// Of a channel over a chunk's cells: its mean in two parts and the sum of squared differences from it.  A sum that 32 bits do
// not hold is kept negative, 2^-200 of it.
struct Moments {
  float mean, rest, squares;
};
__device__ __forceinline__ double mean_of(const Moments &m) { return static_cast<double>(m.mean) + m.rest; }
// Sums over moments take squares as they are and keep their signs: where one is negative they start again (`Again`).
template <bool Again> __device__ __forceinline__ double squares_of(const Moments &m, int &signs) {
  if constexpr (!Again) signs |= __float_as_int(m.squares);
  return Again && m.squares < 0.f ? static_cast<double>(m.squares) * -0x1p200 : m.squares;
}
// partial[sample][chunk][channel].  A thread sums differences from the mean of its first cells, which keeps 32 bits enough
// where a channel's mean is far from zero; threads are joined in 64 bits.
template <typename T, int F>
__global__ __launch_bounds__(kThreads) void group_sums(const T *x, Moments *partial, const Cells s) {
  __shared__ Moments shares[kThreads][8];
  const Place p = place_of(s, blockIdx.x);
  float middle[8] = {}, sum[8] = {}, squares[8] = {}, by[8];
  auto add_up = [&](auto again) {
    const T *at = x + p.at;
    for (int done = 0; done < p.cells; done += kAtOnce, at += kAtOnce * p.stride) {
      Eight<T, F> raw[kAtOnce];
      load_cells(raw, at, p.cells - done, p);
      if (!again && done == 0) {
#pragma unroll
        for (int n = 0; n < kAtOnce; ++n) {
          float v[8];
          raw[n].values(v);
#pragma unroll
          for (int i = 0; i < 8; ++i) middle[i] = fmaf(v[i], 1.f / kAtOnce, middle[i]);
        }
      }
#pragma unroll
      for (int n = 0; n < kAtOnce; ++n) {
        if (done + n >= p.cells) break;
        float v[8];
        raw[n].values(v);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float d = again ? fmaf(v[i], by[i], -middle[i]) : v[i] - middle[i];
          sum[i] += d;
          squares[i] = fmaf(d, d, squares[i]);
        }
      }
    }
  };
  add_up(std::false_type());
  const float each = p.cells ? 1.f / static_cast<float>(p.cells) : 0.f;
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float off = sum[i] * each, left = fmaf(-sum[i], off, squares[i]);
    shares[threadIdx.x][i] = {middle[i], off, left <= 0.f ? 0.f : left};   // (NaN stays)
    most = fmaxf(most, squares[i]);
  }
  if (kFar<T> && !held(most)) {   // channels whose squares are too large once more, values times kDown
    unsigned far = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      by[i] = held(squares[i]) ? 1.f : kDown;
      far |= held(squares[i]) ? 0u : 1u << i;
      middle[i] *= by[i], sum[i] = squares[i] = 0.f;
    }
    add_up(std::true_type());
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (!(far >> i & 1)) continue;
      const float off = sum[i] * each, left = fmaf(-sum[i], off, squares[i]), mean = middle[i] + off;
      shares[threadIdx.x][i] = {mean * 0x1p100f, (middle[i] - mean + off) * 0x1p100f, left < 1e-37f ? -1e-37f : -left};
    }
  }
  __syncthreads();
  const int cells = cells_in(s, blockIdx.x);
  const Rows count(s, cells);
  join_rows<double2>(s, [&](int first, int step, int o, int i, double2 &all) {
    int signs = 0;
    auto add_up = [&](auto again) {
      all = {0., 0.};
      for (int r = first; r < s.tile_rows; r += step) {
        const int n = count.of(r);
        const Moments share = shares[r * s.tile_threads + o][i];
        const double mean = mean_of(share), squares = squares_of<again>(share, signs);
        if (n) all.x += mean * n, all.y += squares + mean * mean * n;
      }
    };
    add_up(std::false_type());
    if (kFar<T> && signs < 0) add_up(std::true_type());
  }, [&](int c, const double2 &all) {
    const double mean = all.x / cells, squares = all.y - all.x * mean;
    const float high = static_cast<float>(mean);
    partial[(sample_of(s) * s.chunks + blockIdx.x) * s.channels + c] = {
        high, static_cast<float>(mean - high), squares > 3.4e38 ? static_cast<float>(squares * -0x1p-200) : squares < 0. ? 0.f : static_cast<float>(squares)};
  });
}

// Two sums over the workgroup, the same for every thread
__device__ __forceinline__ void block_sums(double &a, double &b) {
  __shared__ double lds[2][kThreads / 64];
#pragma unroll
  for (int d = 32; d; d >>= 1) a += __shfl_xor(a, d), b += __shfl_xor(b, d);
  if ((threadIdx.x & 63) == 0) lds[0][threadIdx.x >> 6] = a, lds[1][threadIdx.x >> 6] = b;
  __syncthreads();
  a = b = 0.;
#pragma unroll
  for (int i = 0; i < kThreads / 64; ++i) a += lds[0][i], b += lds[1][i];
  __syncthreads();
}

// A group's mean in two parts and r, from sums over `all` values
__device__ __forceinline__ void put_stats(float *stats, long at, long every, double total, double rest, double all, float eps) {
  const double mean = total / all, left = rest / all - mean * mean, var = left < 0. ? 0. : left;   // (NaN stays)
  stats[at] = static_cast<float>(mean);
  stats[every + at] = static_cast<float>(mean - static_cast<float>(mean));
  stats[2 * every + at] = static_cast<float>(1. / sqrt(var + eps));
}

// A group of a sample: stats[0], [1], [2] = mean, what rounding took from it, r.
__global__ __launch_bounds__(kThreads) void group_finish(const Moments *partial, float *stats, const Cells s, float eps, int batch) {
  const unsigned id = linear_block();
  if (id >= static_cast<unsigned>(batch) * s.groups) return;
  const int b = id / s.groups, g = id % s.groups;
  const Moments *const from = partial + static_cast<long>(b) * s.chunks * s.channels + static_cast<long>(g) * s.group_channels;
  double total = 0., rest = 0.;
  const int across = min(s.group_channels, kThreads), rows = kThreads / across, row = threadIdx.x / across;
  const int chunks = row < rows ? s.chunks : 0;
  int signs = 0;
  auto add_up = [&](auto again) {
    total = rest = 0.;
    for (int c = threadIdx.x % across; c < s.group_channels; c += across)
      for (int first = row; first < chunks; first += kAtOnce * rows) {
        Moments share[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) share[i] = from[static_cast<long>(min(first + i * rows, chunks - 1)) * s.channels + c];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
          const long chunk = first + i * rows;
          const double n = chunk < chunks ? static_cast<double>(min(s.cells, (chunk + 1) * s.each) - chunk * s.each) : 0.;
          const double mean = mean_of(share[i]), squares = squares_of<again>(share[i], signs);
          total += n * mean;
          rest += (chunk < chunks ? squares : 0.) + n * mean * mean;
        }
      }
  };
  add_up(std::false_type());
  if (signs < 0) add_up(std::true_type());
  block_sums(total, rest);
  if (threadIdx.x == 0) put_stats(stats, id, static_cast<long>(batch) * s.groups, total, rest, static_cast<double>(s.cells) * s.group_channels, eps);
}

template <typename T> __device__ __forceinline__ float vector_at(const void *w, bool wide, int c, float absent) {
  return !w ? absent : wide ? static_cast<const float *>(w)[c] : load(static_cast<const T *>(w) + c);
}

template <typename T>
__device__ __forceinline__ void load_vector(float (&to)[8], const void *w, bool wide, const Place &p, float absent) {
#pragma unroll
  for (int i = 0; i < 8; ++i) to[i] = absent;
  if (!w) return;
  if (wide) load8(static_cast<const float *>(w) + p.c, p.left, to);
  else load8(static_cast<const T *>(w) + p.c, p.left, to);
}

// A straight line x a + c in 32 bits, c = shift - mean a in two parts for the a that is used: exact where x is near the mean, however far
// that is from zero.
struct Line {
  float a, high, low;
  __device__ __forceinline__ void set(float mean, float rest, float by, double shift) {
    a = by;
    double c = shift - (static_cast<double>(mean) + rest) * by;
    if (fabs(c) > 3.4e38) a = 0.f, c = shift;   // (values that far from zero beside their deviation are all the same: masked ones; NaN stays)
    high = static_cast<float>(c), low = static_cast<float>(c - high);
  }
  __device__ __forceinline__ float at(float x) const { return fmaf(x, a, high) + low; }
};

// What the channels of a thread need
struct Channels {
  float mean[8], rest[8], r[8], w[8], b[8];
};
template <typename T>
__device__ __forceinline__ void load_channels(Channels &t, const Place &p, const float *stats, const void *weight, const void *bias, bool wide,
                                              const Cells &s) {
  const long every = static_cast<long>(s.batch) * s.groups, first = sample_of(s) * s.groups;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const long at = first + static_cast<unsigned>(min(p.c + i, s.channels - 1)) / static_cast<unsigned>(s.group_channels);
    t.mean[i] = stats[at], t.rest[i] = stats[every + at], t.r[i] = stats[2 * every + at];
  }
  load_vector<T>(t.w, weight, wide, p, 1.f);
  load_vector<T>(t.b, bias, wide, p, 0.f);
}

template <typename T, int Kind, int F>
__global__ __launch_bounds__(kThreads) void group_apply(const T *x, const float *stats, const void *weight, const void *bias, bool wide, T *y,
                                                        const Cells s, float low) {
  const Place p = place_of(s, blockIdx.x);
  if (!p.cells) return;
  Channels t;
  load_channels<T>(t, p, stats, weight, bias, wide, s);
  Line z[8];   // h w + b
#pragma unroll
  for (int i = 0; i < 8; ++i) z[i].set(t.mean[i], t.rest[i], t.r[i] * t.w[i], t.b[i]);
  const T *from = x + p.at;
  T *to = y + p.at;
  for (int done = 0; done < p.cells; done += kAtOnce, from += kAtOnce * p.stride, to += kAtOnce * p.stride) {
    Eight<T, F> raw[kAtOnce];
    load_cells(raw, from, p.cells - done, p);
#pragma unroll
    for (int n = 0; n < kAtOnce; ++n) {
      if (done + n >= p.cells) break;
      float v[8];
      raw[n].values(v);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = Activation<Kind>::value(z[i].at(v[i]), low);
      put_eight<T, F>(to + n * p.stride, p.left, v);
    }
  }
}

// ---- gradients ------------------------------------------------------------------------------------------------------
// Sums of gz and gz h of each channel over a chunk's cells
template <typename T, int Kind, int F>
__global__ __launch_bounds__(kThreads) void group_grad_sums(const T *x, const T *gy, const float *stats, const void *weight, const void *bias,
                                                            bool wide, float2 *partial, const Cells s, float low) {
  __shared__ float2 shares[kThreads][8 + 1];
  const Place p = place_of(s, blockIdx.x);
  float sum[8] = {}, dot[8] = {};
  if (p.cells) {
    Channels t;
    load_channels<T>(t, p, stats, weight, bias, wide, s);
    Line hs[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) hs[i].set(t.mean[i], t.rest[i], t.r[i], 0.);
    const T *at = x + p.at, *gat = gy + p.at;
    for (int done = 0; done < p.cells; done += kAtOnce, at += kAtOnce * p.stride, gat += kAtOnce * p.stride) {
      Eight<T, F> raw[kAtOnce], graw[kAtOnce];
      load_cells(raw, at, p.cells - done, p);
      load_cells(graw, gat, p.cells - done, p);
#pragma unroll
      for (int n = 0; n < kAtOnce; ++n) {
        if (done + n >= p.cells) break;
        float v[8], g[8];
        raw[n].values(v);
        graw[n].values(g);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float h = hs[i].at(v[i]), gz = g[i] * Activation<Kind>::slope(fmaf(h, t.w[i], t.b[i]), low);
          sum[i] += gz;
          dot[i] = fmaf(gz, h, dot[i]);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) shares[threadIdx.x][i] = {sum[i], dot[i]};
  __syncthreads();
  join_rows<float2>(s, [&](int first, int step, int o, int i, float2 &all) {
    for (int r = first; r < s.tile_rows; r += step) {
      const float2 share = shares[r * s.tile_threads + o][i];
      all.x += share.x, all.y += share.y;
    }
  }, [&](int c, const float2 &all) { partial[(sample_of(s) * s.chunks + blockIdx.x) * s.channels + c] = all; });
}

// A group of a sample: means[0], [1] = mean(w gz), mean(w gz h); the channels' sums over all chunks take the first one's place.
template <typename T>
__global__ __launch_bounds__(kThreads) void group_grad_finish(float2 *partial, float *means, const void *weight, bool wide, const Cells s, int batch) {
  __shared__ double2 shares[kThreads];
  const unsigned id = linear_block();
  if (id >= static_cast<unsigned>(batch) * s.groups) return;
  const int b = id / s.groups, g = id % s.groups;
  float2 *const from = partial + static_cast<long>(b) * s.chunks * s.channels + static_cast<long>(g) * s.group_channels;
  double sum = 0., dot = 0.;
  const int across = min(s.group_channels, kThreads), rows = kThreads / across, in = threadIdx.x % across, row = threadIdx.x / across;
  for (int first = 0; first < s.group_channels; first += across) {   // (as many channels at a time as there are threads)
    const int c = first + in;
    double one = 0., two = 0.;
    if (c < s.group_channels && row < rows) {
      for (int chunk = row; chunk < s.chunks; chunk += kAtOnce * rows) {
        float2 share[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) share[i] = from[static_cast<long>(min(chunk + i * rows, s.chunks - 1)) * s.channels + c];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i)
          if (chunk + i * rows < s.chunks) one += share[i].x, two += share[i].y;
      }
    }
    shares[threadIdx.x] = {one, two};
    __syncthreads();
    if (row == 0 && c < s.group_channels) {
      for (int r = 1; r < rows; ++r) one += shares[r * across + in].x, two += shares[r * across + in].y;
      from[c] = {static_cast<float>(one), static_cast<float>(two)};
      const double w = vector_at<T>(weight, wide, g * s.group_channels + c, 1.f);
      sum += w * one, dot += w * two;
    }
    __syncthreads();
  }
  block_sums(sum, dot);
  if (threadIdx.x) return;
  const double all = static_cast<double>(s.cells) * s.group_channels;
  means[id] = static_cast<float>(sum / all);
  means[static_cast<long>(batch) * s.groups + id] = static_cast<float>(dot / all);
}

// Sums of a tile's channels over the samples, in their order: the gradients of weight and bias
struct Vectors {
  const float2 *sums;   // of a sample's channels, `every` from one sample to the next
  void *weight, *bias;
  long every;
  int batch;
};
template <typename T> __device__ __forceinline__ void put_vectors(const Vectors &v, bool wide, int first, int last) {
  __shared__ double2 shares[kThreads];
  const int across = min(last - first, kThreads), in = threadIdx.x % across, team = threadIdx.x / across, teams = kThreads / across;
  for (int c = first + in; c - in < last; c += across) {   // (teams of threads share the samples where there are few channels)
    double sum = 0., dot = 0.;
    if (team < teams && c < last) {
#pragma unroll 4
      for (int b = team; b < v.batch; b += teams) {
        const float2 share = v.sums[b * v.every + c];
        sum += share.x, dot += share.y;
      }
    }
    if (teams > 1) {
      shares[threadIdx.x] = {sum, dot};
      __syncthreads();
      if (team == 0)
        for (int t = 1; t < teams; ++t) sum += shares[t * across + in].x, dot += shares[t * across + in].y;
    }
    if (team || c >= last) continue;
    auto put = [&](void *to, double value) {
      if (!to) return;
      if (wide) static_cast<float *>(to)[c] = static_cast<float>(value);
      else static_cast<T *>(to)[c] = store_cast<T>(static_cast<float>(value));
    };
    put(v.bias, sum);
    put(v.weight, dot);
  }
}
constexpr int kVectorChannels = 16;   // of a workgroup
template <typename T> __global__ __launch_bounds__(kThreads) void group_grad_vectors(const Vectors v, bool wide, int channels) {
  const int first = blockIdx.x * kVectorChannels;
  put_vectors<T>(v, wide, first, min(channels, first + kVectorChannels));
}

template <typename T, int Kind, int F>
__global__ __launch_bounds__(kThreads) void group_grad_apply(const T *x, const T *gy, const float *stats, const float *means, const void *weight,
                                                             const void *bias, bool wide, T *gx, const Vectors sums, const Cells s, float low) {
  if (static_cast<int>(blockIdx.x) == s.chunks) {   // behind the last chunk: a tile's gradients of weight and bias
    if (blockIdx.z == 0) put_vectors<T>(sums, wide, blockIdx.y * kThreads * 8, min(s.channels, static_cast<int>(blockIdx.y + 1) * kThreads * 8));
    return;
  }
  const Place p = place_of(s, blockIdx.x);
  if (!p.cells) return;
  Channels t;
  load_channels<T>(t, p, stats, weight, bias, wide, s);
  float one[8], two[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const long at = sample_of(s) * s.groups + min(p.c + i, s.channels - 1) / s.group_channels;
    one[i] = means[at], two[i] = means[static_cast<long>(s.batch) * s.groups + at];
  }
  Line hs[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) hs[i].set(t.mean[i], t.rest[i], t.r[i], 0.);
  const T *at = x + p.at, *gat = gy + p.at;
  T *to = gx + p.at;
  for (int done = 0; done < p.cells; done += kAtOnce, at += kAtOnce * p.stride, gat += kAtOnce * p.stride, to += kAtOnce * p.stride) {
    Eight<T, F> raw[kAtOnce], graw[kAtOnce];
    load_cells(raw, at, p.cells - done, p);
    load_cells(graw, gat, p.cells - done, p);
#pragma unroll
    for (int n = 0; n < kAtOnce; ++n) {
      if (done + n >= p.cells) break;
      float v[8], g[8];
      raw[n].values(v);
      graw[n].values(g);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float h = hs[i].at(v[i]), gz = g[i] * Activation<Kind>::slope(fmaf(h, t.w[i], t.b[i]), low);
        v[i] = t.r[i] * (fmaf(gz, t.w[i], -one[i]) - h * two[i]);
      }
      put_eight<T, F>(to + n * p.stride, p.left, v);
    }
  }
}

// ---- launches -------------------------------------------------------------------------------------------------------
constexpr long kGroups = 1024;   // workgroups of a launch, about
Cells cells_of(int batch, long cells, int channels, int groups) {
  Cells s{};
  s.cells = cells, s.channels = channels, s.groups = groups, s.group_channels = channels / groups, s.batch = batch;
  const int octets = (channels + 7) / 8, tiles = (octets + kThreads - 1) / kThreads;
  s.tile_threads = std::min(octets, kThreads), s.tile_rows = kThreads / s.tile_threads;
  // about four workgroups per compute unit, of four cells a thread at least, and no more than 256: longer sums in 32 bits lose bits
  const long most = std::max(1L, kGroups / std::max(1L, static_cast<long>(batch) * tiles)), rows = static_cast<long>(kAtOnce) * s.tile_rows;
  s.each = std::max(rows, std::min(256L * s.tile_rows, (cells + most - 1) / most));
  s.each = (s.each + s.tile_rows - 1) / s.tile_rows * s.tile_rows;
  s.chunks = static_cast<int>(std::max(1L, (cells + s.each - 1) / s.each));
  return s;
}
int tiles_of(const Cells &s) { return ((s.channels + 7) / 8 + kThreads - 1) / kThreads; }

// Calls f with the form of the kernels that write `bytes`, as a constant
constexpr size_t kCached = 128 << 20;
template <typename F> void for_form(const Cells &s, size_t bytes, const F &f) {
  if (s.channels < 8) f(std::integral_constant<int, kParts>());
  else if (bytes <= kCached) f(std::integral_constant<int, kWhole>());
  else f(std::integral_constant<int, kWholePast>());
}

constexpr int kMostBatch = 65536;   // (a grid's third dimension)
// Larger batches are taken where the forward pass has the form for small samples.  Its gradients need more registers: where they do not fit,
// the kernels of large samples take a slice of the batch at a time.
int too_many(int batch, long cells, int channels, int groups) {
  MV_REQUIRE(batch < kMostBatch || whole_plan(batch, cells, channels, groups, false).u, "a batch of %d is too large for samples of %ld cells", batch, cells);
  return MV_OK;
}
template <typename F> void for_slices(Cells s, const F &f) {
  for (long first = 0; first < s.batch; first += kMostBatch - 1) {
    s.first = static_cast<int>(first);
    f(s, static_cast<unsigned>(std::min(kMostBatch - 1L, s.batch - first)));
  }
}
int arguments(int batch, long cells, int channels, int groups, int activation, int dtype, int weight_dtype) {
  MV_REQUIRE(dtype == MV_F32 || dtype == MV_F16 || dtype == MV_BF16, "dtype %d is not float32, float16 or bfloat16", dtype);
  MV_REQUIRE(weight_dtype == dtype || weight_dtype == MV_F32, "weight and bias have dtype %d, expected %d or float32", weight_dtype, dtype);
  MV_REQUIRE(batch >= 0 && cells >= 0 && cells <= (1L << 36) && channels > 0 && channels <= (1 << 24), "wrong sizes: a batch of %d, %ld cells of %d channels", batch, cells, channels);
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
  if (whole_plan(batch, cells, channels, groups, false).u) return sizeof(Moments);   // (nothing is put there)
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
  const size_t bytes = dtype_size(dtype) * batch * cells * channels;
  const dim3 grid(s.chunks, tiles_of(s), batch);
  const bool wide = weight_dtype == MV_F32;
  auto *const partial = static_cast<Moments *>(workspace);
  auto *const stat = static_cast<float *>(stats);
  if (const WholePlan whole = whole_plan(batch, cells, channels, groups, false); whole.u)
    return group_norm_whole(whole, x, weight, bias, wide, y, stat, batch, eps, activation, low, dtype, st);
  if (const int status = too_many(batch, cells, channels, groups)) return status;
  MV_FLOATS(dtype, {
    const T *const xt = static_cast<const T *>(x);
    for_form(s, 0, [&](auto form) { group_sums<T, form><<<grid, kThreads, 0, st>>>(xt, partial, s); });
    group_finish<<<linear_grid(static_cast<long>(batch) * groups, kThreads), kThreads, 0, st>>>(partial, stat, s, eps, batch);
    for_activation(activation, [&](auto kind) {
      for_form(s, bytes, [&](auto form) { group_apply<T, kind, form><<<grid, kThreads, 0, st>>>(xt, stat, weight, bias, wide, static_cast<T *>(y), s, low); });
    });
  })
  return check_launch("group_norm");
}

size_t mv_group_norm_backward_workspace_bytes(int batch, int64_t cells, int channels, int groups) {
  if (batch <= 0 || cells <= 0 || channels <= 0 || groups <= 0 || channels % groups) return 0;
  if (whole_plan(batch, cells, channels, groups, true).u) return sizeof(float2) * batch * static_cast<size_t>(channels);   // a sum of each sample's channels
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
  const size_t bytes = dtype_size(dtype) * batch * cells * channels;
  const bool wide = weight_dtype == MV_F32;
  MV_REQUIRE(empty || (x && stats && grad_y), "a tensor is missing");
  MV_REQUIRE(empty || (workspace && workspace_bytes >= mv_group_norm_backward_workspace_bytes(batch, cells, channels, groups)), "the workspace is too small");
  const unsigned tiles = tiles_of(s);
  auto *const partial = static_cast<float2 *>(workspace);
  auto *const means = reinterpret_cast<float *>(static_cast<char *>(workspace) + (empty ? 0 : partial_bytes<float2>(batch, s)));
  auto *const stat = static_cast<const float *>(stats);
  const WholePlan whole = empty ? WholePlan{} : whole_plan(batch, cells, channels, groups, true);
  const Vectors vectors{partial, grad_weight, grad_bias, (whole.u ? 1L : s.chunks) * channels, empty ? 0 : batch};
  const bool wanted = grad_weight || grad_bias, behind = wanted && grad_x && !whole.u && !empty && batch < kMostBatch;   // behind the last chunk
  if (whole.u) {
    if (const int status = group_norm_whole_backward(whole, x, grad_y, stat, weight, bias, wide, grad_x, wanted ? partial : nullptr, batch, activation, low, dtype, st))
      return status;
  } else if (!empty) {
    if (const int status = too_many(batch, cells, channels, groups)) return status;
  }
  MV_FLOATS(dtype, {
    const T *const xt = static_cast<const T *>(x), *const gy = static_cast<const T *>(grad_y);
    if (!empty && !whole.u) {
      for_activation(activation, [&](auto kind) {
        for_form(s, 0, [&](auto form) {
          for_slices(s, [&](const Cells &part, unsigned samples) {
            group_grad_sums<T, kind, form><<<dim3(s.chunks, tiles, samples), kThreads, 0, st>>>(xt, gy, stat, weight, bias, wide, partial, part, low);
          });
        });
      });
      group_grad_finish<T><<<linear_grid(static_cast<long>(batch) * groups, kThreads), kThreads, 0, st>>>(partial, means, weight, wide, s, batch);
      if (grad_x)
        for_activation(activation, [&](auto kind) {
          for_form(s, bytes, [&](auto form) {
            for_slices(s, [&](const Cells &part, unsigned samples) {
              group_grad_apply<T, kind, form><<<dim3(s.chunks + (behind ? 1 : 0), tiles, samples), kThreads, 0, st>>>(xt, gy, stat, means, weight, bias, wide,
                                                                                                                    static_cast<T *>(grad_x), vectors, part, low);
            });
          });
        });
    }
    if (wanted && !behind) group_grad_vectors<T><<<(channels + kVectorChannels - 1) / kVectorChannels, kThreads, 0, st>>>(vectors, wide, channels);
  })
  return check_launch("group_norm backward");
}

}  // extern "C"

// Gradients of cross attention.
//
//   p_ij = 2^(factor q_i.k_j - L_i) = 2^(factor (q_i.k_j - m_i) - l_i)   d_i = do_i.o_i   ds_ij = p_ij (do_i.v_j - d_i)
//   dq_i = scale sum_j ds_ij k_j   dk_j = scale sum_i ds_ij q_i   dv_j = sum_i p_ij do_i
//
// Two kernels form the weights anew, one with a query per lane for dq, one with a key per lane for dk and dv: no atomics,
// the same results every time.  Long sums with few results are split, and the parts added in their order.
//
// Forming the weights twice costs two of seven products, and saves what dq by atomics would: 64 times the scores' count over
// the head's width in additions to memory.  Both kernels are bound by the chain from LDS through products, exponential and
// products again, with two or three wavefronts per SIMD to hide it (registers: sums and operands of a 32 x W tile twice).  In the kernel of
// dk and dv a tile also waits twice for memory, with nothing of its own in between: for the next rows' elements before their
// logarithms are asked for, and for those before the first product (the compiler waits for all loads at both places).
// 2 x 1000 queries over 6912 keys, 8 heads of 64, bf16: dq 77 us, dk and dv 90 us, matrix units 32 and 26 %, vector issue 53
// and 35 % busy.  2 x 32768 queries over 100 keys, 8 heads sharing 2 of 32, float16: 61 and 40 us (+ 7 us for the sums of 128
// splits); 170 MB are read and written for dq.  2 x 2000 over 8192, 8 heads of 128, bf16: 300 and 437 us (four products: 614 TFLOP/s),
// one wavefront per SIMD.
// Registers in memory: 42 of 256 for dk and dv of heads of 96 in 16 bits with the single product, 18 of 168 for those of 32 in bf16 with the
// rest's, up to 32 where there are few keys; 13 of 512 in float32 with 128; 8 of 168 for dq of heads of 64.
#include "attention.hpp"

#include <algorithm>

namespace mv {
namespace {

// float16 has no bits below 2^-24: gradients of weights, which may be far below one, are brought to at most 2^15 by a power
// of two of their own for each column, which follows the largest so far as a softmax's maximum does.
template <typename T> struct Raise {
  static constexpr bool kOn = __is_same(T, __half);
  float by = 0.f;   // 0: nothing but zeros yet
  // of 16 values: scales them, and the sums if the power changes
  template <int N> __device__ __forceinline__ void scale(float (&v)[16], f32x16 (&sum)[N]) {
    if constexpr (kOn) {
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(v[i]));
      top = fmaxf(top, other_half(top));
      if (__ballot(by == 0.f ? top > 0.f : top * by > 32768.f)) {
        float next = by;
        if (by == 0.f ? top > 0.f : top * by > 32768.f)   // to 32 .. 64: room for nine more powers
          next = top < INFINITY ? __builtin_amdgcn_ldexpf(1.f, max(-100, min(100, 6 - __builtin_amdgcn_frexp_expf(top)))) : 1.f;
        const float keep = by == 0.f ? 1.f : next / by;
#pragma unroll
        for (int u = 0; u < N; ++u) sum[u] *= keep;
        by = next;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] *= by;
    }
  }
  __device__ __forceinline__ float back() const { return kOn && by != 0.f ? 1.f / by : 1.f; }
};

template <int N> __device__ __forceinline__ void put_sums(const f32x16 (&o)[N], f32x4 *to, int lane) {
#pragma unroll
  for (int u = 0; u < N; ++u)
#pragma unroll
    for (int i = 0; i < 4; ++i) to[(u * 4 + i) * 64 + lane] = f32x4{o[u][4 * i], o[u][4 * i + 1], o[u][4 * i + 2], o[u][4 * i + 3]};
}
template <int N> __device__ __forceinline__ void add_sums(f32x16 (&o)[N], const f32x4 *from, int lane) {
#pragma unroll
  for (int u = 0; u < N; ++u)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x4 r = from[(u * 4 + i) * 64 + lane];
#pragma unroll
      for (int e = 0; e < 4; ++e) o[u][4 * i + e] += r[e];
    }
}
// One column of the sums, as a row of `dim` elements
template <typename O, int N> __device__ __forceinline__ void store_column(O *row, const f32x16 (&o)[N], int dim, int half) {
#pragma unroll
  for (int u = 0; u < N; ++u) {
    float r[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) r[i] = o[u][i];
    store_results(row, 32 * u, dim, half, r);
  }
}

// Rounding of the weights' gradients to 16 bits for the second product would leave dq with 1.45 - 1.7 times the error of its
// own rounding (they sum to zero over a row, their roundings do not); what it takes away is multiplied too: 1.01 - 1.1 times,
// for a fourth of the kernel's matrix instructions more (62 -> 77 us at 1000 x 6912).  dk and dv sum over queries; theirs is 1.4
// times with the single product, and up to 1.9 where there are few keys (the gradients of two weights are each other's
// negative), few rows, or so few weights that those of a few large ones show: up to 32 keys, 64 rows for a head of keys or 2^20
// weights are multiplied twice as well (1.0 - 1.1 times).  There that costs little (bf16, 8 heads of 64: 6674 queries x 14 keys 19.8 -> 20.1 us,
// 60 x 9000 15.6 -> 17.4; float16, 8 of 32, 32768 x 30 20.8 -> 24.1); it would take 1000 x 6912 from 91 to 126 us.
//
// ---- dq -------------------------------------------------------------------------------------------------------
// As the forward kernel; leaves d_i for the next one.  Without gq that is all.
template <typename T, int W, int WQ>
__global__ __launch_bounds__(256, W > 64 || (sizeof(T) == 4 && W == 64) ? 1 : sizeof(T) == 4 ? 2 : 3) void attend_grad_query(
    AttentionArgs a, const T *out, const T *low, const float *lse, const T *go, T *gq, float *delta, float *part, int row_tiles, int splits) {
  constexpr int DP = stored(W);
  using S = Staging<T, DP, WQ == 1>;
  constexpr int kKeys = S::kRows, kSteps = WQ == 4 ? kKeys / 32 : 1, kOut = W / 32;
  using L = Tile<T, DP, kKeys>;
  __shared__ L tiles[S::kBuffers][2];
  const Place place(a, row_tiles, splits);
  if (!place.in) return;
  const int split = place.split, g = place.g, b = place.b;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
  const int rows = a.heads / a.key_heads * a.queries, row = place.tile * 32 * WQ + (WQ == 4 ? wave * 32 : 0) + (lane & 31);
  const bool live = row < rows;
  const bool any = row - (lane & 31) < rows;   // (a wavefront without rows only brings keys: 2 x 64 queries over 27648 36.4 -> 30.3 us)
  const RowOf at(a, g, live ? row : rows - 1);
  const long at_row = (static_cast<long>(b) * a.queries + at.query) * a.heads + at.head,
             at_l = (static_cast<long>(b) * a.heads + at.head) * a.queries + at.query;
  const float factor = a.factor();

  const T *const k = static_cast<const T *>(a.k) + b * a.ks[0] + g * a.ks[2], *const v = static_cast<const T *>(a.v) + b * a.vs[0] + g * a.vs[2];
  const int length = a.length(b), all_tiles = gq ? (length + kKeys - 1) / kKeys : 0;
  const int first = share(all_tiles, split, splits), last = share(all_tiles, split + 1, splits);
  const int my_key = WQ == 4 ? 0 : 32 * wave;
  Pair<T, DP, kKeys> next(a.ks[1], a.vs[1], a.dim);
  unsigned long long next_use[(kSteps + 1) / 2] = {};
  auto load = [&](int t) {
    next.load(k + t * kKeys * a.ks[1], v + t * kKeys * a.vs[1], length - t * kKeys);
#pragma unroll
    for (int n = 0; n < (kSteps + 1) / 2; ++n) next_use[n] = !any ? 0 : use_bits(a, b, t * kKeys + my_key + 64 * n, kSteps == 1 ? 32 : 64, length);
  };
  auto put = [&](int t) {
    if (a.mask) next.keep(a.mask + b * a.mask_stride + t * kKeys, length - t * kKeys);
    next.put(tiles[t % S::kBuffers]);
  };
  if (first < last) load(first);

  Column<T, W> q, d_o;
  float d_i;
  {
    Column<T, W> o;
    d_o.load(go + at_row * a.dim, live, a.dim, half);
    o.load(out + at_row * a.dim, live, a.dim, half);
    d_i = d_o.dot(o);
    // (o has to be better than its type: with few keys, d_i is as large as the products that it is taken from)
    if (low) o.load(low + at_row * a.dim, live, a.dim, half), d_i += d_o.dot(o);
    d_i += other_half(d_i);
  }
  q.load(static_cast<const T *>(a.q) + b * a.qs[0] + at.query * a.qs[1] + at.head * a.qs[2], live, a.dim, half);
  if (a.scale < 0.f) q.negate();
  RowLog<T> sums;
  if (live) sums.load(a, lse, at_l);
  const float sums_log = sums.log(factor), base = sums.base(factor);
  if (live && split == 0 && half == 0 && (WQ == 4 || wave == 0)) delta[at_l] = d_i;
  if (first < last) put(first);

  f32x16 sum[kOut] = {};
  Raise<T> raise;
  for (int t = first; t < last; ++t) {
    unsigned long long use[(kSteps + 1) / 2];
#pragma unroll
    for (int n = 0; n < (kSteps + 1) / 2; ++n) use[n] = next_use[n];
    __syncthreads();
    if (t + 1 < last) load(t + 1);
    const L &ks = tiles[t % S::kBuffers][0], &vs = tiles[t % S::kBuffers][1];
#pragma unroll
    for (int n = 0; n < kSteps; ++n) {
      const unsigned word = static_cast<unsigned>(use[n / 2] >> (32 * (n % 2)));
      if (!word) continue;
      const int key = my_key + 32 * n;
      f32x16 s = times(ks, key, q, lane);
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] -= base;
      const f32x16 dp = times(vs, key, d_o, lane);
      float ds[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) ds[i] = __builtin_amdgcn_exp2f(fmaf(s[i], factor, -sums_log)) * (dp[i] - d_i);
      if (word != ~0u) {
#pragma unroll
        for (int i = 0; i < 16; ++i) ds[i] = where_bit(word >> (4 * half), result_row(i, 0), ds[i], 0.f);
      }
      raise.scale(ds, sum);
      add_transposed<true>(ks, key, ds, sum, lane);
    }
    if (t + 1 < last) {
      if constexpr (S::kBuffers == 1) __syncthreads();
      put(t + 1);
    }
  }
  const float back = raise.back() * a.scale;
#pragma unroll
  for (int u = 0; u < kOut; ++u) sum[u] *= back;

  if constexpr (WQ == 1) {
    __syncthreads();
    f32x4 *const parts = reinterpret_cast<f32x4 *>(tiles);
    static_assert(sizeof(tiles) >= 3 * kOut * 4 * 64 * sizeof(f32x4), "");
    if (wave) put_sums(sum, parts + (wave - 1) * kOut * 4 * 64, lane);
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int w = 0; w < 3; ++w) add_sums(sum, parts + w * kOut * 4 * 64, lane);
  }
  if (!live || !gq) return;
  if (splits > 1) store_column(part + (static_cast<long>(split) * a.batch * a.queries * a.heads + at_row) * a.dim, sum, a.dim, half);
  else store_column(gq + at_row * a.dim, sum, a.dim, half);
}

// ---- dk, dv -----------------------------------------------------------------------------------------------------
// A key per lane; rows of queries and of output gradients go through LDS.  WK = 4: 32 keys for each wavefront, the same 32
// rows; WK = 1 (few keys): the same 32 keys, each wavefront 32 of 128 rows, joined at the end.  A key that does not count
// spoils nothing but its own column, which is written as zeros.
template <typename T, int W, int WK, bool Fine>
__global__ __launch_bounds__(256, W == 128 || (sizeof(T) == 4 && W > 32) || (W == 96 && Fine) ? 1 : W == 32 && sizeof(T) == 2 ? 3 : 2) void attend_grad_key(
    AttentionArgs a, const float *lse, const float *delta, const T *go, T *gk, T *gv, float *part, int key_tiles, int splits) {
  constexpr int DP = stored(W);
  using S = Staging<T, DP, WK == 1, W != 96>;   // (96: two wavefronts per SIMD, 130 -> 83 us at 1000 x 4000 x 8 heads of 80; 128 would spill)
  constexpr int kRows = S::kRows, kSteps = WK == 4 ? kRows / 32 : 1, kOut = W / 32;
  constexpr float kShift = __is_same(T, __half) ? 15.f : 0.f;   // as in the forward pass
  // Ends of rows at once, but for heads of 33 to 64 channels in 16 bits: with it the compiler keeps 25 registers fewer in use
  // there, and heads of 64 take 100 instead of 90 us (1000 x 6912).
  constexpr bool kEnds = sizeof(T) == 4 || W != 64;
  // Whether rows' largest scores are taken off where there is one to take off, or always (RowLog): taking off zeros, in the shade of the
  // next product, is faster than a branch that the compiler does not schedule across (2 x 2000 over 8192, heads of 128, bf16: 437 and
  // 512 us), but for heads of 32 (2 x 2000 over 27648, float16: 434 and 401 us).
  constexpr bool kAsk = sizeof(T) == 2 && W == 32;
  using L = Tile<T, DP, kRows>;
  __shared__ L tiles[S::kBuffers][2];
  __shared__ float stats[S::kBuffers][3][kRows];   // logarithms, delta, what is taken off the scores first
  __shared__ int far_rows[S::kBuffers][kAsk ? kRows / 32 : 1];
  const Place place(a, key_tiles, splits);
  if (!place.in) return;
  const int split = place.split, g = place.g, b = place.b;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
  const int j = place.tile * 32 * WK + (WK == 4 ? wave * 32 : 0) + (lane & 31), length = a.length(b);
  const bool live = j < a.keys, use = j < length && a.counts(b, j);
  const float factor = a.factor();

  // Rows: all heads of the group, query after query, where a tile holds whole queries; one head after the other where not.
  // Nothing to sum where none of the workgroup's keys counts by its length.
  const int group = a.heads / a.key_heads, inner = kRows % group == 0 ? group : 1, outer = group / inner;
  const int rows = a.queries * inner, per_head = (rows + kRows - 1) / kRows;
  const int all_tiles = place.tile * 32 * WK < length ? outer * per_head : 0;
  const int first = share(all_tiles, split, splits), last = share(all_tiles, split + 1, splits);
  const int my_row = WK == 4 ? 0 : 32 * wave;
  RowLog<T> next_log;
  float next_d = 0.f;
  const long go_row = static_cast<long>(a.heads) * a.dim;
  Pair<T, DP, kRows, kEnds> next(a.qs[1], go_row, a.dim);
  if (inner > 1) next.heads(inner, a.qs[2], a.dim);
  const int my_stat_query = static_cast<unsigned>(threadIdx.x) / static_cast<unsigned>(inner), my_stat_head = threadIdx.x - my_stat_query * inner;
  auto load = [&](int t) {
    const int round = outer > 1 ? t / per_head : 0, row = (t - round * per_head) * kRows, h = g * group + round, left = rows - row;
    const int query = row / inner;
    next.load(static_cast<const T *>(a.q) + b * a.qs[0] + query * a.qs[1] + h * a.qs[2],
              go + (static_cast<long>(b) * a.queries + query) * go_row + static_cast<long>(h) * a.dim, left);
    next_log = RowLog<T>(), next_d = 0.f;
    if (static_cast<int>(threadIdx.x) < min(kRows, left)) {
      const long from = (static_cast<long>(b) * a.heads + h + my_stat_head) * a.queries + query + my_stat_query;
      next_log.load(a, lse, from), next_d = delta[from];
    }
  };
  auto put = [&](int t) {
    next.put(tiles[t % S::kBuffers]);
    if (threadIdx.x < kRows) {
      stats[t % S::kBuffers][0][threadIdx.x] = next_log.log(factor) - kShift;
      stats[t % S::kBuffers][1][threadIdx.x] = next_d;
      stats[t % S::kBuffers][2][threadIdx.x] = next_log.base(factor);
      if constexpr (kAsk) {
        const unsigned long long far = __ballot(next_log.far(factor));
        if ((lane & 31) == 0) far_rows[t % S::kBuffers][threadIdx.x / 32] = static_cast<int>(lane ? far >> 32 : far);
      }
    }
  };
  if (first < last) load(first);
  Column<T, W, kEnds> k, v;
  k.load(static_cast<const T *>(a.k) + b * a.ks[0] + j * a.ks[1] + g * a.ks[2], use, a.dim, half);
  v.load(static_cast<const T *>(a.v) + b * a.vs[0] + j * a.vs[1] + g * a.vs[2], use, a.dim, half);
  if (a.scale < 0.f) k.negate();
  if (first < last) put(first);

  f32x16 dk[kOut] = {}, dv[kOut] = {};
  Raise<T> raise;
  for (int t = first; t < last; ++t) {
    __syncthreads();
    if (t + 1 < last) load(t + 1);
    const L &qs = tiles[t % S::kBuffers][0], &os = tiles[t % S::kBuffers][1];
#pragma unroll
    for (int n = 0; n < kSteps; ++n) {
      const int row = my_row + 32 * n;
      f32x16 s = times(qs, row, k, lane);
      if constexpr (!kAsk) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f32x4 base = *reinterpret_cast<const f32x4 *>(&stats[t % S::kBuffers][2][row + 8 * i + 4 * half]);
#pragma unroll
          for (int e = 0; e < 4; ++e) s[4 * i + e] -= base[e];
        }
      }
      const f32x16 dp = times(os, row, v, lane);
      if constexpr (kAsk) {
        if (__builtin_expect(__builtin_amdgcn_readfirstlane(far_rows[t % S::kBuffers][row / 32]), 0)) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const f32x4 base = *reinterpret_cast<const f32x4 *>(&stats[t % S::kBuffers][2][row + 8 * i + 4 * half]);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[4 * i + e] -= base[e];
          }
        }
      }
      float p[16], ds[16];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x4 l4 = *reinterpret_cast<const f32x4 *>(&stats[t % S::kBuffers][0][row + 8 * i + 4 * half]),
                    d4 = *reinterpret_cast<const f32x4 *>(&stats[t % S::kBuffers][1][row + 8 * i + 4 * half]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          p[4 * i + e] = __builtin_amdgcn_exp2f(fmaf(s[4 * i + e], factor, -l4[e]));
          ds[4 * i + e] = p[4 * i + e] * (dp[4 * i + e] - d4[e]);
        }
      }
      add_transposed<Fine>(os, row, p, dv, lane);
      raise.scale(ds, dk);
      add_transposed<Fine>(qs, row, ds, dk, lane);
    }
    if (t + 1 < last) {
      if constexpr (S::kBuffers == 1) __syncthreads();
      put(t + 1);
    }
  }
  const float down = kShift ? 1.f / 32768.f : 1.f, back = raise.back() * (a.scale * down);
#pragma unroll
  for (int u = 0; u < kOut; ++u) dk[u] *= back, dv[u] *= down;

  if constexpr (WK == 1) {
    f32x4 *const sums = reinterpret_cast<f32x4 *>(tiles);
    static_assert(sizeof(tiles) >= 3 * kOut * 4 * 64 * sizeof(f32x4), "");
    __syncthreads();
    if (wave) put_sums(dk, sums + (wave - 1) * kOut * 4 * 64, lane);
    __syncthreads();
    if (!wave)
#pragma unroll
      for (int w = 0; w < 3; ++w) add_sums(dk, sums + w * kOut * 4 * 64, lane);
    __syncthreads();
    if (wave) put_sums(dv, sums + (wave - 1) * kOut * 4 * 64, lane);
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int w = 0; w < 3; ++w) add_sums(dv, sums + w * kOut * 4 * 64, lane);
  }
  if (!live) return;
  if (!use) {
#pragma unroll
    for (int u = 0; u < kOut; ++u) dk[u] = 0.f, dv[u] = 0.f;
  }
  const long at_row = (static_cast<long>(b) * a.keys + j) * a.key_heads + g, all = static_cast<long>(a.batch) * a.keys * a.key_heads;
  if (splits > 1) {
    store_column(part + (split * all + at_row) * a.dim, dk, a.dim, half);
    store_column(part + ((splits + split) * all + at_row) * a.dim, dv, a.dim, half);
  } else {
    store_column(gk + at_row * a.dim, dk, a.dim, half);
    store_column(gv + at_row * a.dim, dv, a.dim, half);
  }
}

template <typename T> void sum_parts(const float *part, T *out, T *second, long count, int splits, hipStream_t s) {
  const long all = (second ? 2 : 1) * count;
  if (splits >= 16) add_parts<T, 16><<<linear_grid((all + 15) / 16, 256), 256, 0, s>>>(part, out, second, count, splits);
  else add_parts<T, 1><<<linear_grid((all + 255) / 256, 256), 256, 0, s>>>(part, out, second, count, splits);
}

struct BackwardPlan {
  bool few_rows, few_keys, fine;
  int row_tiles, query_splits, key_tiles, key_splits;
};

BackwardPlan backward_plan(const mv_attention_shape *s, int dtype, bool for_query = true) {
  BackwardPlan p;
  const long rows = static_cast<long>(s->heads / s->key_heads) * s->queries, heads = std::max(1L, static_cast<long>(s->batch) * s->key_heads);
  p.few_rows = rows <= 32 && has_few(dtype, s->dim);
  p.few_keys = s->keys <= 32 && has_few(dtype, s->dim);
  p.fine = rows <= 64 || heads * rows * s->keys <= 1 << 20;
  p.row_tiles = static_cast<int>(p.few_rows ? 1 : (rows + 127) / 128);
  p.key_tiles = static_cast<int>(p.few_keys ? 1 : (s->keys + 127L) / 128);
  const int least = dtype == MV_F32 ? 64 : 512;   // keys, or rows, that are worth a split
  const long key_steps = parts_of(s->keys, std::max(least, tile_rows(dtype, s->dim, p.few_rows)));
  // rows as the kernel takes them: those of a group's heads together, or one head after the other
  const int tile = tile_rows(dtype, s->dim, p.few_keys, s->dim <= 64 || s->dim > 96), group = s->heads / s->key_heads, inner = tile % group == 0 ? group : 1;
  const long row_steps = group / inner * parts_of(static_cast<long>(s->queries) * inner, std::max(least, tile));
  // as many workgroups as are resident at a time
  const long for_queries = s->dim <= 64 ? 768 : 256, for_keys = s->dim <= 32 ? 768 : s->dim <= 96 ? 512 : 256;
  p.query_splits = !for_query ? 1 : static_cast<int>(std::max(1L, std::min(for_queries / std::max(1L, p.row_tiles * heads), key_steps)));
  p.key_splits = static_cast<int>(std::max(1L, std::min(for_keys / std::max(1L, p.key_tiles * heads), row_steps)));
  return p;
}

template <typename T, int W>
void launch_backward(const BackwardPlan &p, const AttentionArgs &a, const void *out, const void *low, const float *lse, const void *go, void *gq, void *gk, void *gv,
                     float *delta, float *part, hipStream_t s) {
  const long heads = static_cast<long>(a.batch) * a.key_heads, queries = static_cast<long>(a.batch) * a.queries * a.heads * a.dim,
             keys = heads * a.keys * a.dim;
  const T *const o = static_cast<const T *>(out), *const ol = static_cast<const T *>(low), *const d_o = static_cast<const T *>(go);
  if (queries) {
    const dim3 grid = linear_grid(heads * p.row_tiles * p.query_splits, 256);
    bool done = false;
    if constexpr (kHasFew<T, W>)
      if (p.few_rows) {
        attend_grad_query<T, W, 1><<<grid, 256, 0, s>>>(a, o, ol, lse, d_o, static_cast<T *>(gq), delta, part, p.row_tiles, p.query_splits);
        done = true;
      }
    if (!done) attend_grad_query<T, W, 4><<<grid, 256, 0, s>>>(a, o, ol, lse, d_o, static_cast<T *>(gq), delta, part, p.row_tiles, p.query_splits);
    if (p.query_splits > 1) sum_parts<T>(part, static_cast<T *>(gq), nullptr, queries, p.query_splits, s);
  }
  if (keys && gk) {
    const dim3 grid = linear_grid(heads * p.key_tiles * p.key_splits, 256);
    bool done = false;
    if constexpr (kHasFew<T, W>)
      if (p.few_keys) {
        attend_grad_key<T, W, 1, sizeof(T) == 2><<<grid, 256, 0, s>>>(a, lse, delta, d_o, static_cast<T *>(gk), static_cast<T *>(gv), part, p.key_tiles, p.key_splits);
        done = true;
      }
    if constexpr (sizeof(T) == 2)
      if (!done && p.fine) {
        attend_grad_key<T, W, 4, true><<<grid, 256, 0, s>>>(a, lse, delta, d_o, static_cast<T *>(gk), static_cast<T *>(gv), part, p.key_tiles, p.key_splits);
        done = true;
      }
    if (!done) attend_grad_key<T, W, 4, false><<<grid, 256, 0, s>>>(a, lse, delta, d_o, static_cast<T *>(gk), static_cast<T *>(gv), part, p.key_tiles, p.key_splits);
    if (p.key_splits > 1) sum_parts<T>(part, static_cast<T *>(gk), static_cast<T *>(gv), keys, p.key_splits, s);
  }
}

}  // namespace
}  // namespace mv

using namespace mv;

extern "C" {

size_t mv_cross_attention_backward_workspace_bytes(const mv_attention_shape *s, int dtype) {
  return mv_cross_attention_backward_workspace_bytes_for(s, dtype, 1, 1);
}

size_t mv_cross_attention_backward_workspace_bytes_for(const mv_attention_shape *s, int dtype, int for_query, int for_keys) {
  if (attention_sizes(s, dtype)) return 0;
  const BackwardPlan p = backward_plan(s, dtype, for_query);
  const size_t queries = static_cast<size_t>(s->batch) * s->queries * s->heads, keys = static_cast<size_t>(s->batch) * s->keys * s->key_heads;
  const size_t query_parts = p.query_splits > 1 ? p.query_splits * queries * s->dim : 0,
               key_parts = for_keys && p.key_splits > 1 ? 2 * p.key_splits * keys * s->dim : 0;
  return sizeof(float) * (queries + std::max(query_parts, key_parts));
}

int mv_cross_attention_backward(const void *query, const void *key, const void *value, const void *key_mask,
                                const void *key_lengths, const void *output, const void *output_low, const void *lse, const void *grad_output,
                                void *grad_query, void *grad_key, void *grad_value, const mv_attention_shape *shape,
                                float scale, int dtype, void *workspace, size_t workspace_bytes, void *stream) {
  if (const int status = attention_sizes(shape, dtype)) return status;
  const AttentionArgs a = attention_arguments(shape, query, key, value, key_mask, key_lengths, scale);
  const long rows = static_cast<long>(a.batch) * a.queries * a.heads, columns = static_cast<long>(a.batch) * a.keys * a.key_heads;
  // (a tensor without elements may have any address)
  const bool for_query = rows != 0 && grad_query, for_keys = columns != 0 && (grad_key || grad_value);
  MV_REQUIRE(!for_keys || (grad_key && grad_value), "grad_key and grad_value are wanted as a pair");
  if (!for_query && !for_keys) return MV_OK;
  MV_REQUIRE(rows == 0 || (query && output && lse && grad_output), "a tensor is missing");
  MV_REQUIRE(columns == 0 || (key && value), "a tensor is missing");
  MV_REQUIRE(rows == 0 || (workspace && workspace_bytes >= mv_cross_attention_backward_workspace_bytes_for(shape, dtype, for_query, for_keys)),
             "the workspace is too small");
  const BackwardPlan p = backward_plan(shape, dtype, for_query);
  float *const delta = static_cast<float *>(workspace), *const part = delta + rows;
  const float *const sums = static_cast<const float *>(lse);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  MV_FLOATS(dtype, {
    if (a.dim <= 32) launch_backward<T, 32>(p, a, output, output_low, sums, grad_output, grad_query, grad_key, grad_value, delta, part, s);
    else if (a.dim <= 64) launch_backward<T, 64>(p, a, output, output_low, sums, grad_output, grad_query, grad_key, grad_value, delta, part, s);
    else if (a.dim <= 96) launch_backward<T, 96>(p, a, output, output_low, sums, grad_output, grad_query, grad_key, grad_value, delta, part, s);
    else launch_backward<T, 128>(p, a, output, output_low, sums, grad_output, grad_query, grad_key, grad_value, delta, part, s);
  })
  return check_launch("cross_attention backward");
}

}  // extern "C"

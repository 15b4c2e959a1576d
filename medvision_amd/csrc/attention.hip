// Cross attention of queries over the keys and values of another length: forward.
//
//   s_ij = scale q_i.k_j   p_ij = exp(s_ij - m_i)   l_i = sum_j p_ij   o_i = sum_j p_ij v_j / l_i   L_i = m_i + log l_i
//
// The exponentials are powers of two (log2(e) goes into the scale), running maximum and sums are in 32 bits.
#include "attention.hpp"

#include <algorithm>

namespace mv {
namespace {

// ---- forward -------------------------------------------------------------------------------------------------
// Four wavefronts: WQ = 4, 32 rows each over the same 64 keys at a time; WQ = 1, the same 32 rows, each 32 of 128 keys at a
// time (few rows: their sums are joined at the end).  Scores are formed transposed, a query per lane: maximum and sum of a
// row are those of a lane and of its other half, and the weights are the second product's operand as they stand.
// float16: weights are 2^15 times as large (at most 32768), which keeps those below 2^-14 of the largest from losing bits.
template <typename T, int DP, int WQ>
__global__ __launch_bounds__(256, sizeof(T) == 4 ? (DP == 128 ? 1 : 2) : DP == 128 ? 2 : DP == 64 ? 3 : 4) void attend_kernel(
    AttentionArgs a, T *out, T *low, float *lse, float *part, int row_tiles, int splits) {
  constexpr int kTiles = WQ == 4 ? 2 : 1, kKeys = WQ == 4 ? 64 : 128, kOut = DP / 32;
  constexpr float kShift = sizeof(T) == 2 && __is_same(T, __half) ? 15.f : 0.f;
  using L = Tile<T, DP, kKeys>;
  __shared__ L tiles[2];
  __shared__ float joined[4][2][32];
  L &ks = tiles[0], &vs = tiles[1];
  const int groups = row_tiles * splits * a.batch * a.key_heads;
  unsigned id = linear_block();
  if (id >= static_cast<unsigned>(groups)) return;
  id = xcd_contiguous(id, groups);
  const int tile = id % row_tiles, split = id / row_tiles % splits, g = id / row_tiles / splits % a.key_heads, b = id / row_tiles / splits / a.key_heads;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
  const int rows = a.heads / a.key_heads * a.queries, row = tile * 32 * WQ + (WQ == 4 ? wave * 32 : 0) + (lane & 31);
  const bool live = row < rows;
  const RowOf at(a, g, live ? row : rows - 1);
  const float factor = a.factor();

  Column<T, DP> q;
  q.load(static_cast<const T *>(a.q) + b * a.qs[0] + at.query * a.qs[1] + at.head * a.qs[2], live, a.dim, half);
  if (a.scale < 0.f) q.negate();

  const T *const k = static_cast<const T *>(a.k) + b * a.ks[0] + g * a.ks[2], *const v = static_cast<const T *>(a.v) + b * a.vs[0] + g * a.vs[2];
  const int length = a.length(b), all_tiles = (length + kKeys - 1) / kKeys;
  const int first = static_cast<int>(static_cast<long>(all_tiles) * split / splits), last = static_cast<int>(static_cast<long>(all_tiles) * (split + 1) / splits);
  const int my_key = WQ == 4 ? 0 : 32 * wave;   // of a tile
  Carry<T, DP, kKeys, 256> next_k, next_v;
  unsigned long long next_use = 0;
  auto load = [&](int t) {
    const auto use = [&](int j) { return a.counts(b, j); };
    next_k.load(threadIdx.x, t * kKeys, length, a.dim, [&](int j) { return k + j * a.ks[1]; }, use);
    next_v.load(threadIdx.x, t * kKeys, length, a.dim, [&](int j) { return v + j * a.vs[1]; }, use);
    const int j = t * kKeys + my_key + lane;
    next_use = __ballot(j < length && (WQ == 4 || lane < 32) && a.counts(b, min(j, length - 1)));
  };

  float m = -INFINITY, l = 0.f;
  f32x16 o[kOut] = {};
  if (first < last) load(first);
  for (int t = first; t < last; ++t) {
    if (t > first) __syncthreads();   // the last tile has been read
    next_k.put(threadIdx.x, ks);
    next_v.put(threadIdx.x, vs);
    const unsigned long long use = next_use;
    __syncthreads();
    if (t + 1 < last) load(t + 1);
    if (!use) continue;
    f32x16 s[kTiles];
#pragma unroll
    for (int n = 0; n < kTiles; ++n) s[n] = times(ks, my_key + 32 * n, q, lane);
    if (use != (kTiles == 2 ? ~0ull : 0xffffffffull)) {
#pragma unroll
      for (int n = 0; n < kTiles; ++n) {
        const unsigned word = static_cast<unsigned>(use >> (32 * n)) >> (4 * half);
#pragma unroll
        for (int i = 0; i < 16; ++i) s[n][i] = word >> result_row(i, 0) & 1 ? s[n][i] : -INFINITY;
      }
    }
    float top = s[0][0];
#pragma unroll
    for (int n = 0; n < kTiles; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, s[n][i]);
    top = fmaxf(m, fmaxf(top, other_half(top)));
    const float base = top == -INFINITY ? 0.f : top;
    if (__ballot(top > m)) {   // (no row's maximum has grown: nothing to scale)
      const float keep = __builtin_amdgcn_exp2f((m - base) * factor);
      l *= keep;
#pragma unroll
      for (int u = 0; u < kOut; ++u) o[u] *= keep;
      m = top;
    }
    const float shift = fmaf(base, -factor, kShift);
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
      float p[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        // (float32: the difference first, so that the largest weight is one to the last bit)
        const float x = sizeof(T) == 4 ? (s[n][i] - base) * factor : fmaf(s[n][i], factor, shift);
        l += p[i] = __builtin_amdgcn_exp2f(x);
      }
      add_transposed(vs, my_key + 32 * n, p, o, lane);
    }
  }
  l += other_half(l);

  if constexpr (WQ == 1) {   // four sums of the same rows
    __syncthreads();
    f32x4 *const sums = reinterpret_cast<f32x4 *>(tiles);
    static_assert(sizeof(tiles) >= 3 * kOut * 4 * 64 * sizeof(f32x4), "");
    if (half == 0) joined[wave][0][lane] = m, joined[wave][1][lane] = l;
    __syncthreads();
    float top = -INFINITY, total = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) top = fmaxf(top, joined[w][0][lane & 31]);
    const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int w = 0; w < 4; ++w) total += joined[w][1][lane & 31] * __builtin_amdgcn_exp2f((joined[w][0][lane & 31] - base) * factor);
    const float keep = __builtin_amdgcn_exp2f((m - base) * factor);
#pragma unroll
    for (int u = 0; u < kOut; ++u) o[u] *= keep;
    if (wave) {
#pragma unroll
      for (int u = 0; u < kOut; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          sums[(((wave - 1) * kOut + u) * 4 + i) * 64 + lane] = f32x4{o[u][4 * i], o[u][4 * i + 1], o[u][4 * i + 2], o[u][4 * i + 3]};
    }
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int u = 0; u < kOut; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int w = 0; w < 3; ++w) {
          const f32x4 r = sums[((w * kOut + u) * 4 + i) * 64 + lane];
#pragma unroll
          for (int e = 0; e < 4; ++e) o[u][4 * i + e] += r[e];
        }
    m = top, l = total;
  }
  if (!live) return;
  const long at_row = (static_cast<long>(b) * a.queries + at.query) * a.heads + at.head;   // of the output
  if (splits > 1) {   // the sums as they are, maximum and sum beside them
    const long all = static_cast<long>(a.batch) * a.queries * a.heads;
    float *const to = part + (split * all + at_row) * a.dim;
#pragma unroll
    for (int u = 0; u < kOut; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) store_quad(to, 32 * u + 8 * i + 4 * half, a.dim, o[u][4 * i], o[u][4 * i + 1], o[u][4 * i + 2], o[u][4 * i + 3]);
    if (half == 0) {
      float *const stats = part + splits * all * a.dim + (split * all + at_row) * 2;
      stats[0] = m, stats[1] = l;
    }
    return;
  }
  const float inverse = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int u = 0; u < kOut; ++u)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = 32 * u + 8 * i + 4 * half;
      float r[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) r[e] = o[u][4 * i + e] * inverse;
      store_quad(out + at_row * a.dim, d, a.dim, r[0], r[1], r[2], r[3]);
      if (low) store_quad(low + at_row * a.dim, d, a.dim, rest_of<T>(r[0]), rest_of<T>(r[1]), rest_of<T>(r[2]), rest_of<T>(r[3]));
    }
  if (lse && half == 0)
    lse[(static_cast<long>(b) * a.heads + at.head) * a.queries + at.query] = l == 0.f ? -INFINITY : fmaf(m, factor, __log2f(l) - kShift);
}

// The splits' sums of one row: a wavefront.
template <typename T>
__global__ __launch_bounds__(256) void join_splits(AttentionArgs a, const float *part, T *out, T *low, float *lse, int splits, float shift) {
  const long all = static_cast<long>(a.batch) * a.queries * a.heads, row = static_cast<long>(linear_block()) * 4 + (threadIdx.x >> 6);
  if (row >= all) return;
  const int lane = threadIdx.x & 63;
  const float *const stats = part + splits * all * a.dim, factor = a.factor();
  float top = -INFINITY, l = 0.f, o[2] = {};
  for (int s = 0; s < splits; ++s) top = fmaxf(top, stats[(s * all + row) * 2]);
  const float base = top == -INFINITY ? 0.f : top;
  for (int s = 0; s < splits; ++s) {
    const float keep = __builtin_amdgcn_exp2f((stats[(s * all + row) * 2] - base) * factor);
    l += keep * stats[(s * all + row) * 2 + 1];
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (lane + 64 * e < a.dim) o[e] += keep * part[(s * all + row) * a.dim + lane + 64 * e];
  }
  const float inverse = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int e = 0; e < 2; ++e)
    if (lane + 64 * e < a.dim) {
      const long to = row * a.dim + lane + 64 * e;
      out[to] = store_cast<T>(o[e] * inverse);
      if (low) low[to] = store_cast<T>(rest_of<T>(o[e] * inverse));
    }
  if (lse && lane == 0) {
    const int h = row % a.heads, i = row / a.heads % a.queries, b = row / a.heads / a.queries;
    lse[(static_cast<long>(b) * a.heads + h) * a.queries + i] = l == 0.f ? -INFINITY : fmaf(top, factor, __log2f(l) - shift);
  }
}

struct ForwardPlan {
  bool few;
  int row_tiles, splits;
};

ForwardPlan forward_plan(const mv_attention_shape *s) {
  const long rows = static_cast<long>(s->heads / s->key_heads) * s->queries;
  const bool few = rows <= 32;
  const long row_tiles = few ? 1 : (rows + 127) / 128, groups = std::max(1L, row_tiles * s->batch * s->key_heads);
  const long tiles = few ? (s->keys + 127L) / 128 : (s->keys + 63L) / 64;
  return {few, static_cast<int>(row_tiles), static_cast<int>(std::max(1L, std::min(512 / groups, tiles / 4)))};
}

template <typename T, int DP>
void launch_forward(const ForwardPlan &p, const AttentionArgs &a, void *out, void *low, float *lse, float *part, hipStream_t s) {
  const long groups = static_cast<long>(p.row_tiles) * p.splits * a.batch * a.key_heads;
  const dim3 grid = linear_grid(groups, 256);
  if (p.few) attend_kernel<T, DP, 1><<<grid, 256, 0, s>>>(a, static_cast<T *>(out), static_cast<T *>(low), lse, part, p.row_tiles, p.splits);
  else attend_kernel<T, DP, 4><<<grid, 256, 0, s>>>(a, static_cast<T *>(out), static_cast<T *>(low), lse, part, p.row_tiles, p.splits);
}

}  // namespace
}  // namespace mv

using namespace mv;

extern "C" {

size_t mv_cross_attention_forward_workspace_bytes(const mv_attention_shape *s, int dtype) {
  if (attention_sizes(s, dtype)) return 0;
  const ForwardPlan p = forward_plan(s);
  return p.splits > 1 ? sizeof(float) * p.splits * s->batch * static_cast<size_t>(s->queries) * s->heads * (s->dim + 2) : 0;
}

int mv_cross_attention_forward(const void *query, const void *key, const void *value, const void *key_mask,
                               const void *key_lengths, void *output, void *output_low, void *lse, const mv_attention_shape *shape,
                               float scale, int dtype, void *workspace, size_t workspace_bytes, void *stream) {
  if (const int status = attention_sizes(shape, dtype)) return status;
  const AttentionArgs a = attention_arguments(shape, query, key, value, key_mask, key_lengths, scale);
  const long rows = static_cast<long>(a.batch) * a.queries * a.heads;
  if (rows == 0) return MV_OK;
  MV_REQUIRE(query && output && (a.keys == 0 || (key && value)), "a tensor is missing");
  ForwardPlan p = forward_plan(shape);
  if (p.splits > 1 && (!workspace || workspace_bytes < mv_cross_attention_forward_workspace_bytes(shape, dtype))) p.splits = 1;
  float *const part = static_cast<float *>(workspace), *const sums = static_cast<float *>(lse);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  MV_FLOATS(dtype, {
    if (a.dim <= 32) launch_forward<T, 32>(p, a, output, output_low, sums, part, s);
    else if (a.dim <= 64) launch_forward<T, 64>(p, a, output, output_low, sums, part, s);
    else launch_forward<T, 128>(p, a, output, output_low, sums, part, s);
    if (p.splits > 1)
      join_splits<T><<<linear_grid((rows + 3) / 4, 256), 256, 0, s>>>(a, part, static_cast<T *>(output), static_cast<T *>(output_low), sums, p.splits, dtype == MV_F16 ? 15.f : 0.f);
  })
  return check_launch("cross_attention");
}

}  // extern "C"

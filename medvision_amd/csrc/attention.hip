// Cross attention of queries over the keys and values of another length: forward.
//
//   s_ij = scale q_i.k_j   p_ij = exp(s_ij - m_i)   l_i = sum_j p_ij   o_i = sum_j p_ij v_j / l_i   L_i = m_i + log l_i
//
// The exponentials are powers of two (log2(e) goes into the scale), running maximum and sums are in 32 bits.
#include "attention.hpp"

#include <algorithm>

namespace mv {
namespace {

// log2 of a row's sum of weights beside the largest one, and the largest score (RowLog takes them)
__device__ __forceinline__ void put_log(const AttentionArgs &a, float *lse, long at, float m, float l, float shift) {
  lse[at] = l == 0.f ? -INFINITY : __log2f(l) - shift;
  lse[static_cast<long>(a.batch) * a.heads * a.queries + at] = l == 0.f ? 0.f : m;
}

// ---- forward -------------------------------------------------------------------------------------------------
// Four wavefronts: WQ = 4, 32 rows each over the same 64 keys at a time; WQ = 1, the same 32 rows, each 32 of 128 keys at a
// time (few rows: their sums are joined at the end).  Scores are formed transposed, a query per lane: maximum and sum of a
// row are those of a lane and of its other half, and the weights are the second product's operand as they stand.
// float16: weights are 2^15 times as large (at most 32768), which keeps those below 2^-14 of the largest from losing bits.
// The weights are rounded to the values' type for the second product (a matrix instruction has one type), maximum, sum and
// output stay in 32 bits: the error against 64 bits is 1.1 - 1.3 times that of rounding the output alone.
//
// Heads of 32: of a score, 6.6 issue slots are vector instructions (two of them the exponential), two matrix instructions.  2 x 2000
// queries x 8 heads over 27648 keys of 32, float16: 221 us with the join of four splits = 4.0e12 scores/s, vector units 73 % and
// matrix units 22 % busy.  The rest is waiting: the columns' loads may be outstanding where the loop starts, so the compiler waits for
// all loads in front of each tile's first product, the next tile's among them, and only other wavefronts cover those.  Heads of 64
// (2 x 1000 over 6912, bf16): 50 us, vector units 46 %, matrix units 23 %; of 128 (2 x 2000 over 8192): 163 us = 820 TFLOP/s,
// two wavefronts per SIMD, LDS 45 %, matrix units 35 %.  One query per sample reads the keys once: 4 samples of 32768 keys, 16 heads over 4 of
// 64 channels: 25 us + 5 us for the join of 32 splits (134 MB at full length: 5.3 TB/s).  float32 on its own matrix instructions:
// 2 x 2000 over 4096, 8 heads of 64: 297 us = 113 of 154 TFLOP/s, matrix units 71 % busy.  2 x 32768 queries over 100 keys, 8 heads sharing
// 2 of 32, float16, with the output's low bits: 39 us, 102 MB (keys held in LDS over several tiles of rows, with the next queries
// on their way, were a tenth slower: that takes 167 registers instead of 128).
// Few rows: 128 keys at a time, with heads of more than 64 channels in all 256 registers of two wavefronts per SIMD, and 17 (96) or
// 40 (128) of them in memory; 13 in float32 with 64 (heads of 64 in 16 bits run on two wavefronts too, not on three).  2 x 8 queries
// over 32768 keys, 8 heads of 64 26 us, of 96 44, of 128 63 to 68: 134, 201 and 268 MB, 5.1, 4.6 and 4.2 TB/s.
template <typename T, int W, int WQ>
__global__ __launch_bounds__(256, sizeof(T) == 4 ? (W > 64 ? 1 : 2) : W > 64 ? 2 : W == 64 ? 3 : 4) void attend_kernel(
    AttentionArgs a, T *out, T *low, float *lse, float *part, int row_tiles, int splits) {
  constexpr int DP = stored(W);
  using S = Staging<T, DP, WQ == 1>;
  constexpr int kTiles = WQ == 4 && S::kRows >= 64 ? 2 : 1, kKeys = S::kRows, kSteps = WQ == 4 ? kKeys / (32 * kTiles) : 1, kOut = W / 32;
  constexpr float kShift = __is_same(T, __half) ? 15.f : 0.f;
  using L = Tile<T, DP, kKeys>;
  __shared__ L tiles[S::kBuffers][2];
  __shared__ float joined[4][2][32];
  const Place place(a, row_tiles, splits);
  if (!place.in) return;
  const int split = place.split, g = place.g, b = place.b;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
  const int rows = a.heads / a.key_heads * a.queries, row = place.tile * 32 * WQ + (WQ == 4 ? wave * 32 : 0) + (lane & 31);
  const bool live = row < rows;
  const bool any = row - (lane & 31) < rows;   // (a wavefront without rows only brings keys: 2 x 64 queries over 27648 24.7 -> 19.5 us)
  const RowOf at(a, g, live ? row : rows - 1);
  const float factor = a.factor();

  const T *const k = static_cast<const T *>(a.k) + b * a.ks[0] + g * a.ks[2], *const v = static_cast<const T *>(a.v) + b * a.vs[0] + g * a.vs[2];
  const int length = a.length(b), all_tiles = (length + kKeys - 1) / kKeys;
  const int first = share(all_tiles, split, splits), last = share(all_tiles, split + 1, splits);
  const int my_key = WQ == 4 ? 0 : 32 * wave;   // of a tile
  Pair<T, DP, kKeys> next(a.ks[1], a.vs[1], a.dim);
  unsigned long long next_use[kSteps] = {};
  auto load = [&](int t) {
    next.load(k + t * kKeys * a.ks[1], v + t * kKeys * a.vs[1], length - t * kKeys);
#pragma unroll
    for (int n = 0; n < kSteps; ++n) next_use[n] = !any ? 0 : use_bits(a, b, t * kKeys + my_key + 32 * kTiles * n, 32 * kTiles, length);
  };
  auto put = [&](int t) {
    if (a.mask) next.keep(a.mask + b * a.mask_stride + t * kKeys, length - t * kKeys);
    next.put(tiles[t % S::kBuffers]);
  };
  if (first < last) load(first);
  Column<T, W> q;
  q.load(static_cast<const T *>(a.q) + b * a.qs[0] + at.query * a.qs[1] + at.head * a.qs[2], live, a.dim, half);
  if (a.scale < 0.f) q.negate();
  if (first < last) put(first);

  float m = -INFINITY, l = 0.f;
  bool far = false;
  f32x16 o[kOut] = {};
  for (int t = first; t < last; ++t) {
    unsigned long long use[kSteps];
#pragma unroll
    for (int n = 0; n < kSteps; ++n) use[n] = next_use[n];
    __syncthreads();   // this tile is there, and the one before it has been read
    if (t + 1 < last) load(t + 1);
    const L &ks = tiles[t % S::kBuffers][0], &vs = tiles[t % S::kBuffers][1];
#pragma unroll
    for (int step = 0; step < kSteps; ++step) {
      if (!use[step]) continue;
      const int key = my_key + 32 * kTiles * step;
      f32x16 s[kTiles];
#pragma unroll
      for (int n = 0; n < kTiles; ++n) s[n] = times(ks, key + 32 * n, q, lane);
      if (use[step] != (kTiles == 2 ? ~0ull : 0xffffffffull)) {
#pragma unroll
        for (int n = 0; n < kTiles; ++n) {
          const unsigned word = static_cast<unsigned>(use[step] >> (32 * n)) >> (4 * half);
#pragma unroll
          for (int i = 0; i < 16; ++i) s[n][i] = where_bit(word, result_row(i, 0), s[n][i], -INFINITY);
        }
      }
      float top = s[0][0];
#pragma unroll
      for (int n = 0; n < kTiles; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, s[n][i]);
      top = fmaxf(m, fmaxf(top, other_half(top)));
      float base = top == -INFINITY ? 0.f : top;
      if (__ballot(top > m)) {   // (no row's maximum has grown: nothing to scale)
        far = sizeof(T) == 2 && __ballot(fabsf(base) * factor > kFar);
        const float keep = __builtin_amdgcn_exp2f((m - base) * factor);
        l *= keep;
#pragma unroll
        for (int u = 0; u < kOut; ++u) o[u] *= keep;
        m = top;
      }
      if (__builtin_expect(far, false)) {   // (the difference first)
#pragma unroll
        for (int n = 0; n < kTiles; ++n) s[n] -= base;
        base = 0.f;
      }
      const float shift = fmaf(base, -factor, kShift);
#pragma unroll
      for (int n = 0; n < kTiles; ++n) {
        float p[16], sum[4];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          // (float32: the difference first, so that the largest weight is one to the last bit)
          const float x = sizeof(T) == 4 ? (s[n][i] - base) * factor : fmaf(s[n][i], factor, shift);
          p[i] = __builtin_amdgcn_exp2f(x);
          sum[i % 4] = i < 4 ? p[i] : sum[i % 4] + p[i];
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        add_transposed(vs, key + 32 * n, p, o, lane);
      }
    }
    if (t + 1 < last) {
      if constexpr (S::kBuffers == 1) __syncthreads();
      put(t + 1);
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
  for (int u = 0; u < kOut; ++u) {
    float r[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) r[i] = o[u][i] * inverse;
    store_results(out + at_row * a.dim, 32 * u, a.dim, half, r);
    if (low) {
#pragma unroll
      for (int i = 0; i < 16; ++i) r[i] = rest_of<T>(r[i]);
      store_results(low + at_row * a.dim, 32 * u, a.dim, half, r);
    }
  }
  if (lse && half == 0) put_log(a, lse, (static_cast<long>(b) * a.heads + at.head) * a.queries + at.query, m, l, kShift);
}

// The splits' sums.  Many splits (few rows): a workgroup for a row, whose wavefronts take turns at the splits.
template <typename T>
__global__ __launch_bounds__(256) void join_many(AttentionArgs a, const float *part, T *out, T *low, float *lse, int splits, float shift) {
  __shared__ float sums[4][1 + kMostDim];
  const long all = static_cast<long>(a.batch) * a.queries * a.heads, row = linear_block();
  if (row >= all) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const float *const stats = part + splits * all * a.dim, factor = a.factor();
  float top = -INFINITY, l = 0.f, o[2] = {};
  for (int s = lane; s < splits; s += 64) top = fmaxf(top, stats[(s * all + row) * 2]);
#pragma unroll
  for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
  const float base = top == -INFINITY ? 0.f : top;
#pragma unroll 4
  for (int s = wave; s < splits; s += 4) {
    const float keep = __builtin_amdgcn_exp2f((stats[(s * all + row) * 2] - base) * factor);
    l += keep * stats[(s * all + row) * 2 + 1];
#pragma unroll
    for (int e = 0; e < 2; ++e) o[e] += keep * part[(s * all + row) * a.dim + min(lane + 64 * e, a.dim - 1)];
  }
  sums[wave][lane] = o[0], sums[wave][64 + lane] = o[1];
  if (lane == 0) sums[wave][kMostDim] = l;
  __syncthreads();
  l = ((sums[0][kMostDim] + sums[1][kMostDim]) + sums[2][kMostDim]) + sums[3][kMostDim];
  const float inverse = l == 0.f ? 0.f : 1.f / l;
  const int d = threadIdx.x;
  if (d < a.dim) {
    const float v = (((sums[0][d] + sums[1][d]) + sums[2][d]) + sums[3][d]) * inverse;
    out[row * a.dim + d] = store_cast<T>(v);
    if (low) low[row * a.dim + d] = store_cast<T>(rest_of<T>(v));
  }
  if (lse && threadIdx.x == 0) put_log(a, lse, a.log_at(row), top, l, shift);
}

// Few splits: four neighbouring elements of a row per thread.
template <typename T>
__global__ __launch_bounds__(256) void join_few(AttentionArgs a, const float *part, T *out, T *low, float *lse, int splits, float shift) {
  const int quads = (a.dim + 3) / 4;
  const long all = static_cast<long>(a.batch) * a.queries * a.heads, at = static_cast<long>(linear_block()) * 256 + threadIdx.x, row = at / quads;
  if (row >= all) return;
  const int d = static_cast<int>(at - row * quads) * 4;
  const float *const stats = part + splits * all * a.dim, factor = a.factor();
  float top = -INFINITY, l = 0.f, o[4] = {};
  for (int s = 0; s < splits; ++s) top = fmaxf(top, stats[(s * all + row) * 2]);
  const float base = top == -INFINITY ? 0.f : top;
#pragma unroll 4
  for (int s = 0; s < splits; ++s) {
    const float keep = __builtin_amdgcn_exp2f((stats[(s * all + row) * 2] - base) * factor);
    l += keep * stats[(s * all + row) * 2 + 1];
    const float *const from = part + (s * all + row) * a.dim;
    if (d + 4 <= a.dim) {
      const f32x4 r = reinterpret_cast<const Loose<f32x4, 4> *>(from + d)->v;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += keep * r[e];
    } else {
#pragma unroll
      for (int e = 0; e < 3; ++e) o[e] += keep * from[min(d + e, a.dim - 1)];
    }
  }
  const float inverse = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] *= inverse;
  store_quad(out + row * a.dim, d, a.dim, o[0], o[1], o[2], o[3]);
  if (low) store_quad(low + row * a.dim, d, a.dim, rest_of<T>(o[0]), rest_of<T>(o[1]), rest_of<T>(o[2]), rest_of<T>(o[3]));
  if (lse && d == 0) put_log(a, lse, a.log_at(row), top, l, shift);
}

// Four wavefronts have 128 rows, or the 32 rows that there are.  Keys are split until every resident workgroup has work
// (registers and LDS: four per compute unit for heads of 32, three of 64, two beyond), but into no fewer than 512 (the join
// is a launch, 3 - 4 us, and 512 keys take about as long), 64 in float32 (16 us): one query over 343 keys 7.1 us in one piece,
// 10.7 in two.
struct ForwardPlan {
  bool few;
  int row_tiles, splits;
};

ForwardPlan forward_plan(const mv_attention_shape *s, int dtype) {
  const long rows = static_cast<long>(s->heads / s->key_heads) * s->queries;
  const bool few = rows <= 32 && has_few(dtype, s->dim);
  const long row_tiles = few ? 1 : (rows + 127) / 128, groups = std::max(1L, row_tiles * s->batch * s->key_heads);
  const long shares = parts_of(s->keys, std::max(dtype == MV_F32 ? 64 : 512, tile_rows(dtype, s->dim, few)));   // the least worth a split
  return {few, static_cast<int>(row_tiles), static_cast<int>(std::max(1L, std::min((s->dim <= 32 ? 1024 : s->dim <= 64 && !few ? 768 : 512) / groups, shares)))};
}

template <typename T, int W>
void launch_forward(const ForwardPlan &p, const AttentionArgs &a, void *out, void *low, float *lse, float *part, hipStream_t s) {
  const long groups = static_cast<long>(p.row_tiles) * p.splits * a.batch * a.key_heads;
  const dim3 grid = linear_grid(groups, 256);
  if constexpr (kHasFew<T, W>)
    if (p.few) {
      attend_kernel<T, W, 1><<<grid, 256, 0, s>>>(a, static_cast<T *>(out), static_cast<T *>(low), lse, part, p.row_tiles, p.splits);
      return;
    }
  attend_kernel<T, W, 4><<<grid, 256, 0, s>>>(a, static_cast<T *>(out), static_cast<T *>(low), lse, part, p.row_tiles, p.splits);
}

}  // namespace
}  // namespace mv

using namespace mv;

extern "C" {

size_t mv_cross_attention_forward_workspace_bytes(const mv_attention_shape *s, int dtype) {
  if (attention_sizes(s, dtype)) return 0;
  const ForwardPlan p = forward_plan(s, dtype);
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
  ForwardPlan p = forward_plan(shape, dtype);
  if (p.splits > 1 && (!workspace || workspace_bytes < mv_cross_attention_forward_workspace_bytes(shape, dtype))) p.splits = 1;
  float *const part = static_cast<float *>(workspace), *const sums = static_cast<float *>(lse);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  MV_FLOATS(dtype, {
    if (a.dim <= 32) launch_forward<T, 32>(p, a, output, output_low, sums, part, s);
    else if (a.dim <= 64) launch_forward<T, 64>(p, a, output, output_low, sums, part, s);
    else if (a.dim <= 96) launch_forward<T, 96>(p, a, output, output_low, sums, part, s);
    else launch_forward<T, 128>(p, a, output, output_low, sums, part, s);
    const float shift = dtype == MV_F16 ? 15.f : 0.f;
    T *const o = static_cast<T *>(output), *const ol = static_cast<T *>(output_low);
    // (a workgroup for a row also where those are few: 16 rows of 32 channels, 8 splits 4.0 us, 7.2 with quads of elements)
    if (p.splits > (rows <= 256 ? 4 : 8)) join_many<T><<<linear_grid(rows, 256), 256, 0, s>>>(a, part, o, ol, sums, p.splits, shift);
    else if (p.splits > 1) join_few<T><<<linear_grid((rows * ((a.dim + 3) / 4) + 255) / 256, 256), 256, 0, s>>>(a, part, o, ol, sums, p.splits, shift);
  })
  return check_launch("cross_attention");
}

}  // extern "C"

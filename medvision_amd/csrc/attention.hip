// Cross attention of queries over the keys and values of another length, forward and backward.
//
//   s_ij = scale q_i.k_j   p_ij = exp(s_ij - L_i), L_i = log sum_j exp(s_ij)   o_i = sum_j p_ij v_j
//   d_i = do_i.o_i   ds_ij = p_ij (do_i.v_j - d_i)
//   dq_i = scale sum_j ds_ij k_j   dk_j = scale sum_i ds_ij q_i   dv_j = sum_i p_ij do_i
//
// The exponentials are powers of two (log2(e) goes into the scale), running maximum and sums are in 32 bits.
#include "rows.hpp"

namespace mv {
namespace {

constexpr int kMostDim = 128;
constexpr float kLog2e = 1.44269504088896f;

struct AttentionArgs {
  const void *q, *k, *v;
  const unsigned char *mask;
  const int *lengths;
  int batch, queries, keys, heads, key_heads, dim;
  long qs[3], ks[3], vs[3], mask_stride;
  float scale;
  __device__ __forceinline__ int length(int b) const { return lengths ? min(max(lengths[b], 0), keys) : keys; }
  __device__ __forceinline__ bool counts(int b, int j) const { return !mask || mask[b * mask_stride + j]; }
};

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
  return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v = fmaxf(v, __shfl_xor(v, d));
  return v;
}

template <typename T> __device__ __forceinline__ float dot(const T *row, const float *with, int dim) {
  float s = 0.f;
  for (int d = 0; d < dim; d += 8) {
    float v[8];
    load8(row + d, dim - d, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) s += v[i] * with[d + i];   // (`with` is filled with zeros up to kMostDim)
  }
  return s;
}

// One wavefront per query and head: keys by lane for the scores, columns by lane for the sums.
template <typename T>
__global__ __launch_bounds__(256) void attend_kernel(AttentionArgs a, T *out, float *lse) {
  __shared__ float rows[4][kMostDim];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long at = static_cast<long>(linear_block()) * 4 + wave;
  const bool live = at < static_cast<long>(a.batch) * a.queries * a.heads;
  const int h = at % a.heads, i = at / a.heads % a.queries, b = at / a.heads / a.queries, g = h / (a.heads / a.key_heads);
  const T *q = static_cast<const T *>(a.q) + b * a.qs[0] + i * a.qs[1] + h * a.qs[2];
  const T *k = static_cast<const T *>(a.k) + b * a.ks[0] + g * a.ks[2], *v = static_cast<const T *>(a.v) + b * a.vs[0] + g * a.vs[2];
  float *const row = rows[wave];
  for (int d = lane; d < kMostDim; d += 64) row[d] = live && d < a.dim ? load(q + d) : 0.f;
  __syncthreads();
  if (!live) return;
  const int length = a.length(b);
  float m = -INFINITY, l = 0.f, o[2] = {};
  for (int j0 = 0; j0 < length; j0 += 64) {
    const int j = j0 + lane;
    const bool use = j < length && a.counts(b, j);
    const float s = use ? dot(k + j * a.ks[1], row, a.dim) * (a.scale * kLog2e) : -INFINITY;
    const unsigned long long all = __ballot(use);
    if (!all) continue;
    const float top = fmaxf(m, wave_max(s)), base = top == -INFINITY ? 0.f : top;
    const float p = use ? exp2f(s - base) : 0.f, keep = exp2f(m - base);
    l = l * keep + wave_sum(p);
    o[0] *= keep, o[1] *= keep;
    for (int jj = 0; jj < 64; ++jj) {
      if (!(all >> jj & 1)) continue;
      const float pj = __shfl(p, jj);
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (lane + 64 * e < a.dim) o[e] += pj * load(v + (j0 + jj) * a.vs[1] + lane + 64 * e);
    }
    m = top;
  }
  const float inverse = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int e = 0; e < 2; ++e)
    if (lane + 64 * e < a.dim) out[at * a.dim + lane + 64 * e] = store_cast<T>(o[e] * inverse);
  if (lse && lane == 0) lse[(static_cast<long>(b) * a.heads + h) * a.queries + i] = l == 0.f ? -INFINITY : m + log2f(l);
}

// One wavefront per query and head; leaves d_i for the kernel below.
template <typename T>
__global__ __launch_bounds__(256) void attend_grad_query(AttentionArgs a, const T *out, const float *lse, const T *go, T *gq, float *delta) {
  __shared__ float rows[4][2][kMostDim];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long at = static_cast<long>(linear_block()) * 4 + wave;
  const bool live = at < static_cast<long>(a.batch) * a.queries * a.heads;
  const int h = at % a.heads, i = at / a.heads % a.queries, b = at / a.heads / a.queries, g = h / (a.heads / a.key_heads);
  const T *q = static_cast<const T *>(a.q) + b * a.qs[0] + i * a.qs[1] + h * a.qs[2];
  const T *k = static_cast<const T *>(a.k) + b * a.ks[0] + g * a.ks[2], *v = static_cast<const T *>(a.v) + b * a.vs[0] + g * a.vs[2];
  float d_i = 0.f;
  for (int d = lane; d < kMostDim; d += 64) {
    const bool in = live && d < a.dim;
    rows[wave][0][d] = in ? load(q + d) : 0.f;
    rows[wave][1][d] = in ? load(go + at * a.dim + d) : 0.f;
    if (in) d_i += rows[wave][1][d] * load(out + at * a.dim + d);
  }
  d_i = wave_sum(d_i);
  __syncthreads();
  if (!live) return;
  const long at_l = (static_cast<long>(b) * a.heads + h) * a.queries + i;
  const float L = lse[at_l];
  if (lane == 0) delta[at_l] = d_i;
  const int length = L == -INFINITY ? 0 : a.length(b);
  float sum[2] = {};
  for (int j0 = 0; j0 < length; j0 += 64) {
    const int j = j0 + lane;
    const bool use = j < length && a.counts(b, j);
    float ds = 0.f;
    if (use) {
      const float p = exp2f(dot(k + j * a.ks[1], rows[wave][0], a.dim) * (a.scale * kLog2e) - L);
      ds = p * (dot(v + j * a.vs[1], rows[wave][1], a.dim) - d_i);
    }
    const unsigned long long all = __ballot(use);
    for (int jj = 0; jj < 64; ++jj) {
      if (!(all >> jj & 1)) continue;
      const float dj = __shfl(ds, jj);
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (lane + 64 * e < a.dim) sum[e] += dj * load(k + (j0 + jj) * a.ks[1] + lane + 64 * e);
    }
  }
#pragma unroll
  for (int e = 0; e < 2; ++e)
    if (lane + 64 * e < a.dim) gq[at * a.dim + lane + 64 * e] = store_cast<T>(sum[e] * a.scale);
}

// One wavefront per key and key head, over the queries of all heads that share it.
template <typename T>
__global__ __launch_bounds__(256) void attend_grad_key(AttentionArgs a, const float *lse, const float *delta, const T *go, T *gk, T *gv) {
  __shared__ float rows[4][2][kMostDim];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long at = static_cast<long>(linear_block()) * 4 + wave;
  const bool live = at < static_cast<long>(a.batch) * a.keys * a.key_heads;
  const int g = at % a.key_heads, j = at / a.key_heads % a.keys, b = at / a.key_heads / a.keys, group = a.heads / a.key_heads;
  const bool use = live && j < a.length(b) && a.counts(b, j);
  for (int d = lane; d < kMostDim; d += 64) {
    const bool in = use && d < a.dim;
    rows[wave][0][d] = in ? load(static_cast<const T *>(a.k) + b * a.ks[0] + j * a.ks[1] + g * a.ks[2] + d) : 0.f;
    rows[wave][1][d] = in ? load(static_cast<const T *>(a.v) + b * a.vs[0] + j * a.vs[1] + g * a.vs[2] + d) : 0.f;
  }
  __syncthreads();
  if (!live) return;
  float sk[2] = {}, sv[2] = {};
  for (int h = g * group; use && h < (g + 1) * group; ++h) {
    const T *q = static_cast<const T *>(a.q) + b * a.qs[0] + h * a.qs[2];
    for (int i0 = 0; i0 < a.queries; i0 += 64) {
      const int i = i0 + lane, count = min(64, a.queries - i0);
      float p = 0.f, ds = 0.f;
      if (i < a.queries) {
        const long at_l = (static_cast<long>(b) * a.heads + h) * a.queries + i, at_o = (static_cast<long>(b) * a.queries + i) * a.heads + h;
        p = exp2f(dot(q + i * a.qs[1], rows[wave][0], a.dim) * (a.scale * kLog2e) - lse[at_l]);
        ds = p * (dot(go + at_o * a.dim, rows[wave][1], a.dim) - delta[at_l]);
      }
      for (int ii = 0; ii < count; ++ii) {
        const float pi = __shfl(p, ii), di = __shfl(ds, ii);
        const long at_o = (static_cast<long>(b) * a.queries + i0 + ii) * a.heads + h;
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (lane + 64 * e < a.dim) {
            sv[e] += pi * load(go + at_o * a.dim + lane + 64 * e);
            sk[e] += di * load(q + (i0 + ii) * a.qs[1] + lane + 64 * e);
          }
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 2; ++e)
    if (lane + 64 * e < a.dim) {
      gk[at * a.dim + lane + 64 * e] = store_cast<T>(sk[e] * a.scale);
      gv[at * a.dim + lane + 64 * e] = store_cast<T>(sv[e]);
    }
}

#define MV_FLOATS(dtype, ...)                                                                                    \
  switch (dtype) {                                                                                               \
    case MV_F32: { using T = float; __VA_ARGS__; break; }                                                        \
    case MV_F16: { using T = __half; __VA_ARGS__; break; }                                                       \
    case MV_BF16: { using T = __hip_bfloat16; __VA_ARGS__; break; }                                              \
    default: return ::mv::fail(MV_INVALID_ARGUMENT, "dtype %d is not float32, float16 or bfloat16", (int)(dtype)); \
  }

int attention_sizes(const mv_attention_shape *s, int dtype) {
  MV_REQUIRE(s, "the shape is missing");
  MV_REQUIRE(dtype == MV_F32 || dtype == MV_F16 || dtype == MV_BF16, "dtype %d is not float32, float16 or bfloat16", dtype);
  MV_REQUIRE(s->batch >= 0 && s->queries >= 0 && s->keys >= 0, "wrong sizes: batch %d, %d queries, %d keys", s->batch, s->queries, s->keys);
  MV_REQUIRE(s->key_heads > 0 && s->heads > 0 && s->heads % s->key_heads == 0, "%d heads cannot share %d heads of keys", s->heads, s->key_heads);
  MV_REQUIRE(s->dim > 0 && s->dim <= kMostDim, "heads of %d channels: 1 to %d are possible", s->dim, kMostDim);
  return MV_OK;
}

AttentionArgs arguments(const mv_attention_shape *s, const void *q, const void *k, const void *v, const void *mask, const void *lengths, float scale) {
  AttentionArgs a{q, k, v, static_cast<const unsigned char *>(mask), static_cast<const int *>(lengths), s->batch, s->queries, s->keys,
                  s->heads, s->key_heads, s->dim, {}, {}, {}, static_cast<long>(s->mask_stride), scale};
  for (int i = 0; i < 3; ++i) a.qs[i] = s->q_strides[i], a.ks[i] = s->k_strides[i], a.vs[i] = s->v_strides[i];
  return a;
}

}  // namespace
}  // namespace mv

using namespace mv;

extern "C" {

size_t mv_cross_attention_forward_workspace_bytes(const mv_attention_shape *shape, int dtype) { return 0; }

size_t mv_cross_attention_backward_workspace_bytes(const mv_attention_shape *s, int dtype) {
  if (attention_sizes(s, dtype)) return 0;
  return sizeof(float) * s->batch * s->heads * static_cast<size_t>(s->queries);
}

int mv_cross_attention_forward(const void *query, const void *key, const void *value, const void *key_mask,
                               const void *key_lengths, void *output, void *lse, const mv_attention_shape *shape,
                               float scale, int dtype, void *workspace, size_t workspace_bytes, void *stream) {
  if (const int status = attention_sizes(shape, dtype)) return status;
  const AttentionArgs a = arguments(shape, query, key, value, key_mask, key_lengths, scale);
  const long rows = static_cast<long>(a.batch) * a.queries * a.heads;
  if (rows == 0) return MV_OK;
  MV_REQUIRE(query && output && (a.keys == 0 || (key && value)), "a tensor is missing");
  MV_FLOATS(dtype, attend_kernel<T><<<linear_grid((rows + 3) / 4, 256), 256, 0, static_cast<hipStream_t>(stream)>>>(
      a, static_cast<T *>(output), static_cast<float *>(lse)))
  return check_launch("cross_attention");
}

int mv_cross_attention_backward(const void *query, const void *key, const void *value, const void *key_mask,
                                const void *key_lengths, const void *output, const void *lse, const void *grad_output,
                                void *grad_query, void *grad_key, void *grad_value, const mv_attention_shape *shape,
                                float scale, int dtype, void *workspace, size_t workspace_bytes, void *stream) {
  if (const int status = attention_sizes(shape, dtype)) return status;
  const AttentionArgs a = arguments(shape, query, key, value, key_mask, key_lengths, scale);
  const long rows = static_cast<long>(a.batch) * a.queries * a.heads, columns = static_cast<long>(a.batch) * a.keys * a.key_heads;
  MV_REQUIRE(rows == 0 || (query && output && lse && grad_output && grad_query), "a tensor is missing");
  MV_REQUIRE(columns == 0 || (key && value && grad_key && grad_value), "a tensor is missing");
  MV_REQUIRE(rows == 0 || (workspace && workspace_bytes >= mv_cross_attention_backward_workspace_bytes(shape, dtype)), "the workspace is too small");
  float *const delta = static_cast<float *>(workspace);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  MV_FLOATS(dtype, {
    if (rows > 0)
      attend_grad_query<T><<<linear_grid((rows + 3) / 4, 256), 256, 0, s>>>(a, static_cast<const T *>(output), static_cast<const float *>(lse),
          static_cast<const T *>(grad_output), static_cast<T *>(grad_query), delta);
    if (columns > 0)
      attend_grad_key<T><<<linear_grid((columns + 3) / 4, 256), 256, 0, s>>>(a, static_cast<const float *>(lse), delta,
          static_cast<const T *>(grad_output), static_cast<T *>(grad_key), static_cast<T *>(grad_value));
  })
  return check_launch("cross_attention backward");
}

}  // extern "C"

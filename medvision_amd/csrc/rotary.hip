// Rotary positions on several axes: pair p of a head's channels is turned by the angle  sum over axes a of  place[a] f[a, p].
//
//   (x1, x2) -> (x1 cos - x2 sin, x1 sin + x2 cos); the gradient is turned back
//
// A pair is (p, pairs + p), or (2p, 2p + 1).  Angles are formed in 64 bits (32 would lose the turn of far places) in
// quarters of a turn, whose whole part swaps sine and cosine and whose rest goes through a polynomial in 32 bits.  A
// workgroup forms the angles of its rows once for all heads, in LDS.  Bound by memory: one pass over it.
#include "rows.hpp"

#include <algorithm>

namespace mv {
namespace {

constexpr int kThreads = 256;
constexpr int kMostDim = 1024, kMostAxes = 8;
constexpr int kTable = 4096;   // angles of a workgroup at most

struct Rotary {
  mv_rotary_shape of;
  int block_rows, row_blocks;
};

__device__ __forceinline__ double place_at(const void *p, int kind, long at) {
  return kind == MV_F32 ? static_cast<const float *>(p)[at] : kind == MV_F64 ? static_cast<const double *>(p)[at] : static_cast<const int *>(p)[at];
}

// Cosine and sine of q quarters of a turn; polynomials of least relative error for |r| <= 1/2: 6e-11 and 3e-9, roundings in 32 bits on top
__device__ __forceinline__ float2 turn(double q) {
  const double whole = rint(q);
  const float r = static_cast<float>(q - whole), u = r * r;
  float s = -4.6016578870e-03f, c = 9.0336297626e-04f;
  s = fmaf(s, u, 7.9680032768e-02f);
  s = fmaf(s, u, -6.4596346023e-01f);
  s = fmaf(s, u, 1.5707963217f) * r;
  c = fmaf(c, u, -2.0859936028e-02f);
  c = fmaf(c, u, 2.5366918260e-01f);
  c = fmaf(c, u, -1.2337005396f);
  c = fmaf(c, u, 1.f);
  const int quarter = static_cast<int>(whole - 4. * floor(0.25 * whole));   // 0 .. 3
  const float a = quarter & 1 ? s : c, b = quarter & 1 ? c : s;
  return {quarter == 1 || quarter == 2 ? -a : a, quarter >= 2 ? -b : b};
}

template <typename T, bool Neighbours>
__global__ __launch_bounds__(kThreads) void rotary(const T *x, const void *places, int place_kind, const double *frequencies, T *y,
                                                   const Rotary k, bool back) {
  extern __shared__ float2 table[];
  const mv_rotary_shape &s = k.of;
  const unsigned id = linear_block();
  if (id >= static_cast<unsigned>(s.batch) * k.row_blocks) return;
  const int b = id / k.row_blocks;
  const int first = (id - b * k.row_blocks) * k.block_rows, rows = min(k.block_rows, s.rows - first);
  const int pairs = s.pairs;
  for (int e = threadIdx.x; e < rows * pairs; e += kThreads) {
    const int row = e / pairs, p = e - row * pairs;
    const long at = b * s.place_strides[0] + (first + row) * s.place_strides[1];
    double angle = 0.;
    for (int a = 0; a < s.axes; ++a) angle = fma(place_at(places, place_kind, at + a * s.place_strides[2]), frequencies[a * pairs + p], angle);
    float2 t = turn(angle * 0.63661977236758134);   // 2 / pi
    if (back) t.y = -t.y;
    table[e] = t;
  }
  __syncthreads();
  const int turned = (Neighbours ? 2 * pairs + 7 : pairs + 7) / 8, kept = (s.dim - 2 * pairs + 7) / 8, pieces = turned + kept;
  for (int e = threadIdx.x; e < rows * s.heads * pieces; e += kThreads) {
    const int line = e / pieces, o = e - line * pieces, row = line / s.heads, head = line - row * s.heads;
    const T *const from = x + b * s.x_strides[0] + (first + row) * s.x_strides[1] + head * s.x_strides[2];
    T *const to = y + ((static_cast<long>(b) * s.rows + first + row) * s.heads + head) * s.dim;
    if (o >= turned) {   // channels that stay
      const int c = 2 * pairs + (o - turned) * 8;
      float v[8];
      load8(from + c, s.dim - c, v);
      store8(to + c, s.dim - c, v);
      continue;
    }
    if constexpr (Neighbours) {
      const int c = o * 8, left = 2 * pairs - c;
      float v[8];
      load8(from + c, left, v);
      const float2 *const t = table + row * pairs + o * 4;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (2 * i >= left) break;
        const float2 cs = t[i];
        const float one = v[2 * i], two = v[2 * i + 1];
        v[2 * i] = fmaf(one, cs.x, -(two * cs.y));
        v[2 * i + 1] = fmaf(one, cs.y, two * cs.x);
      }
      store8(to + c, left, v);
    } else {
      const int c = o * 8, left = pairs - c;
      float one[8], two[8];
      load8(from + c, left, one);
      load8(from + pairs + c, left, two);
      const float2 *const t = table + row * pairs + c;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (i >= left) break;
        const float2 cs = t[i];
        const float was = one[i];
        one[i] = fmaf(was, cs.x, -(two[i] * cs.y));
        two[i] = fmaf(was, cs.y, two[i] * cs.x);
      }
      store8(to + c, left, one);
      store8(to + pairs + c, left, two);
    }
  }
}

}  // namespace
}  // namespace mv

using namespace mv;

extern "C" int mv_rotary_positions(const void *x, const void *places, const void *frequencies, void *y, const mv_rotary_shape *shape,
                                   int neighbours, int back, int dtype, int place_dtype, void *stream) {
  MV_REQUIRE(shape, "the shape is missing");
  const mv_rotary_shape &s = *shape;
  MV_REQUIRE(dtype == MV_F32 || dtype == MV_F16 || dtype == MV_BF16, "dtype %d is not float32, float16 or bfloat16", dtype);
  MV_REQUIRE(place_dtype == MV_F32 || place_dtype == MV_F64 || place_dtype == MV_I32, "places have dtype %d, expected float32, float64 or int32", place_dtype);
  MV_REQUIRE(s.batch >= 0 && s.rows >= 0 && s.heads >= 0 && s.dim >= 1 && s.dim <= kMostDim && s.axes >= 1 && s.axes <= kMostAxes,
             "wrong sizes: a batch of %d, %d rows, %d heads of %d channels (1 to %d), %d axes (1 to %d)", s.batch, s.rows, s.heads, s.dim, kMostDim, s.axes, kMostAxes);
  MV_REQUIRE(s.pairs >= 0 && 2 * s.pairs <= s.dim, "%d pairs of %d channels", s.pairs, s.dim);
  if (s.batch == 0 || s.rows == 0 || s.heads == 0) return MV_OK;
  MV_REQUIRE(x && y && (s.pairs == 0 || (places && frequencies)), "a tensor is missing");
  Rotary k{s, 0, 0};
  const long row = static_cast<long>(s.heads) * s.dim;
  MV_REQUIRE(row < (1L << 31), "rows of %d heads of %d channels are too long", s.heads, s.dim);
  // 8192 elements a workgroup: four times eight for a thread
  k.block_rows = static_cast<int>(std::max(1L, std::min({8192L / row, 64L, kTable / std::max(1L, static_cast<long>(s.pairs)), static_cast<long>(s.rows)})));
  k.row_blocks = (s.rows + k.block_rows - 1) / k.block_rows;
  const long blocks = static_cast<long>(s.batch) * k.row_blocks;
  MV_REQUIRE(blocks < (1L << 32), "too many rows: %d in a batch of %d", s.rows, s.batch);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const size_t lds = sizeof(float2) * k.block_rows * s.pairs;
  MV_FLOATS(dtype, {
    const auto kernel = neighbours ? rotary<T, true> : rotary<T, false>;
    kernel<<<linear_grid(blocks, kThreads), kThreads, lds, st>>>(static_cast<const T *>(x), places, place_dtype, static_cast<const double *>(frequencies),
                                                                static_cast<T *>(y), k, back != 0);
  })
  return check_launch("rotary_positions");
}

// Rotary positions on several axes: pair p of a head's channels is turned by the angle  sum over axes a of  place[a] f[a, p].
//
//   (x1, x2) -> (x1 cos - x2 sin, x1 sin + x2 cos); the gradient is turned back
//
// A pair is (p, pairs + p), or (2p, 2p + 1).  Angles are formed in 64 bits (32 would lose the turn of far places) in
// quarters of a turn, whose whole part swaps sine and cosine and whose rest goes through a polynomial in 32 bits.  A
// workgroup forms the angles of its rows once for all heads, in LDS.  Bound by memory, one pass over it: 2 x 32768 rows of 8 heads of 64 in
// bf16 with 30 pairs 29 - 32 us (134 MB, 4.2 - 4.6 TB/s; with 32 pairs 31), 2 x 27648 of 8 heads
// of 32 in float16, neighbours, 15 us a way (57 MB).
#include "rows.hpp"

#include <algorithm>

namespace mv {
namespace {

constexpr int kThreads = 256;
constexpr int kMostDim = 1024, kMostAxes = 8;
constexpr int kTable = 4096;   // angles of a workgroup at most

// a / b for 0 <= a < 2^31 with a multiplication: m = floor(2^(31 + s) / b) + 1, 2^(s - 1) < b <= 2^s (exact: a m / 2^(31 + s) is off
// by less than 1 / b)
struct Divisor {
  unsigned by, m;
  int shift;
  explicit Divisor(unsigned b) : by(b), shift(0) {
    while ((1ul << shift) < b) ++shift;
    m = static_cast<unsigned>((1ul << (31 + shift)) / b + 1);
  }
  __device__ __forceinline__ unsigned of(unsigned a) const { return static_cast<unsigned>((static_cast<unsigned long>(a) * m) >> (31 + shift)); }
};

struct Rotary {
  mv_rotary_shape of;
  int block_rows, row_blocks, pieces, kept, unit;   // pieces of eight pairs (channels) of a head; units of the channels that stay
  int kept_here;   // units that go with a head's first pieces (0: by themselves)
  Divisor by_pairs, by_pieces, by_heads, by_kept;
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

template <typename T, int N> __device__ __forceinline__ void copy_unit(const T *from, T *to) {
  typedef unsigned char bytes __attribute__((ext_vector_type(N * sizeof(T) > 16 ? 16 : N * sizeof(T))));
#pragma unroll
  for (unsigned i = 0; i < N * sizeof(T); i += sizeof(bytes))
    reinterpret_cast<Loose<bytes, sizeof(T)> *>(reinterpret_cast<char *>(to) + i)->v = reinterpret_cast<const Loose<bytes, sizeof(T)> *>(reinterpret_cast<const char *>(from) + i)->v;
}

// Up to 16 bytes of channels that stay
template <typename T> struct Stays {
  u32x4 bits;
  template <typename V> static __device__ __forceinline__ Loose<V, sizeof(T)> *at(T *p) { return reinterpret_cast<Loose<V, sizeof(T)> *>(p); }
  template <typename V> static __device__ __forceinline__ const Loose<V, sizeof(T)> *at(const T *p) { return reinterpret_cast<const Loose<V, sizeof(T)> *>(p); }
  __device__ __forceinline__ void load(int unit, const T *p) {
    switch (unit * sizeof(T)) {
      case 16: bits = at<u32x4>(p)->v; break;
      case 8: { const u32x2 v = at<u32x2>(p)->v; bits = {v[0], v[1], 0u, 0u}; break; }
      case 4: bits = {at<unsigned>(p)->v, 0u, 0u, 0u}; break;
      default: bits = {at<unsigned short>(p)->v, 0u, 0u, 0u};
    }
  }
  __device__ __forceinline__ void store(int unit, T *p) const {
    switch (unit * sizeof(T)) {
      case 16: at<u32x4>(p)->v = bits; break;
      case 8: at<u32x2>(p)->v = u32x2{bits[0], bits[1]}; break;
      case 4: at<unsigned>(p)->v = bits[0]; break;
      default: at<unsigned short>(p)->v = static_cast<unsigned short>(bits[0]);
    }
  }
};

// Cosines and sines of a workgroup's rows
__device__ __forceinline__ void form_table(float2 *table, const void *places, int place_kind, const double *frequencies, const Rotary &k, int b, int first,
                                           int rows, bool back) {
  const mv_rotary_shape &s = k.of;
  for (int e = threadIdx.x; e < rows * s.pairs; e += kThreads) {
    const int row = k.by_pairs.of(e), p = e - row * s.pairs;
    const long at = b * s.place_strides[0] + (first + row) * s.place_strides[1];
    double place[4], f[4];   // (axes that do not exist: the last one again)
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const int axis = min(a, s.axes - 1);
      place[a] = place_at(places, place_kind, at + axis * s.place_strides[2]), f[a] = frequencies[axis * s.pairs + p];
    }
    double angle = place[0] * f[0];
#pragma unroll
    for (int a = 1; a < 4; ++a) angle = a < s.axes ? fma(place[a], f[a], angle) : angle;
    for (int a = 4; a < s.axes; ++a) angle = fma(place_at(places, place_kind, at + a * s.place_strides[2]), frequencies[a * s.pairs + p], angle);
    float2 t = turn(angle * 0.63661977236758134);   // 2 / pi
    if (back) t.y = -t.y;
    table[e] = t;
  }
}

// Up to eight pairs: (one[i], two[i]), or neighbours in one[].
template <bool Neighbours> __device__ __forceinline__ void turn_piece(const float2 *t, int left, float (&one)[8], float (&two)[8]) {
#pragma unroll
  for (int i = 0; i < (Neighbours ? 4 : 8); ++i) {
    if ((Neighbours ? 2 * i : i) >= left) break;
    const float2 cs = t[i];
    float &a = one[Neighbours ? 2 * i : i], &b = Neighbours ? one[2 * i + 1] : two[i];
    const float was = a;
    a = fmaf(was, cs.x, -(b * cs.y));
    b = fmaf(was, cs.y, b * cs.x);
  }
}

// Pieces are of eight pairs (neighbours: of eight channels).  The last one of a head starts earlier than its place where the pairs
// do not fill it: what two pieces have in common is formed twice, with the same results, instead of an element at a time.  Channels
// that stay go with a head's first pieces where there are no more units of them: by themselves, later, they cost 37 instead of 31 us.
// A thread's first piece is on its way while the angles are formed.
template <typename T, bool Neighbours>
__global__ __launch_bounds__(kThreads) void rotary(const T *x, const void *places, int place_kind, const double *frequencies, T *y,
                                                   const Rotary k, bool back) {
  extern __shared__ float2 table[];
  const mv_rotary_shape &s = k.of;
  const unsigned id = linear_block();
  if (id >= static_cast<unsigned>(s.batch) * k.row_blocks) return;
  const int b = id / k.row_blocks;
  const int first = (id - b * k.row_blocks) * k.block_rows, rows = min(k.block_rows, s.rows - first), pairs = s.pairs;
  const T *const from = x + b * s.x_strides[0] + first * s.x_strides[1];
  T *const to = y + (static_cast<long>(b) * s.rows + first) * s.heads * s.dim;
  const int lines = rows * s.heads, width = Neighbours ? 2 * pairs : pairs, items = lines * k.pieces;
  struct Piece {
    int row, c, own;
    long from, to;
  };
  auto piece_of = [&](int e) {
    const int line = k.by_pieces.of(e), row = k.by_heads.of(line), own = e - line * k.pieces, c = max(0, min(own * 8, width - 8));
    return Piece{row, c, own, row * s.x_strides[1] + (line - row * s.heads) * s.x_strides[2] + c, static_cast<long>(line) * s.dim + c};
  };
  if (width >= 8) {
    bool formed = false;
    for (int e = threadIdx.x; !formed || e < items; e += kThreads) {
      const Piece p = piece_of(min(e, items - 1));
      Raw<T> one, two;
      one.load(from + p.from);
      if (!Neighbours) two.load(from + p.from + pairs);
      const bool keeps = p.own < k.kept_here;
      const int after = 2 * pairs - p.c + p.own * k.unit;   // from the piece to its unit of the channels that stay
      Stays<T> stays;
      if (keeps) stays.load(k.unit, from + p.from + after);
      if (!formed) {
        form_table(table, places, place_kind, frequencies, k, b, first, rows, back);
        __syncthreads();
        formed = true;
      }
      if (e >= items) break;
      float v[8], w[8];
      one.values(v);
      if (!Neighbours) two.values(w);
      turn_piece<Neighbours>(table + p.row * pairs + (Neighbours ? p.c / 2 : p.c), 8, v, w);
      store8(to + p.to, 8, v);
      if (!Neighbours) store8(to + p.to + pairs, 8, w);
      if (keeps) stays.store(k.unit, to + p.to + after);
    }
    if (k.kept_here) return;
  } else {   // heads of few pairs
    form_table(table, places, place_kind, frequencies, k, b, first, rows, back);
    __syncthreads();
    for (int e = threadIdx.x; e < items; e += kThreads) {
      const Piece p = piece_of(e);
      float v[8], w[8];
      load8(from + p.from, width, v);
      if (!Neighbours) load8(from + p.from + pairs, width, w);
      turn_piece<Neighbours>(table + p.row * pairs, width, v, w);
      store8(to + p.to, width, v);
      if (!Neighbours) store8(to + p.to + pairs, width, w);
    }
  }
  for (int e = threadIdx.x; e < lines * k.kept; e += kThreads) {   // channels that stay
    const int line = k.by_kept.of(e), row = k.by_heads.of(line), head = line - row * s.heads, c = 2 * pairs + (e - line * k.kept) * k.unit;
    const T *const here = from + row * s.x_strides[1] + head * s.x_strides[2] + c;
    T *const there = to + static_cast<long>(line) * s.dim + c;
    switch (k.unit) {
      case 8: copy_unit<T, 8>(here, there); break;
      case 4: copy_unit<T, 4>(here, there); break;
      case 2: copy_unit<T, 2>(here, there); break;
      default: *there = *here;
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
  MV_REQUIRE(s.pairs >= 0 && s.pairs <= s.dim / 2, "%d pairs of %d channels", s.pairs, s.dim);
  if (s.batch == 0 || s.rows == 0 || s.heads == 0) return MV_OK;
  MV_REQUIRE(x && y && (s.pairs == 0 || (places && frequencies)), "a tensor is missing");
  const long row = static_cast<long>(s.heads) * s.dim;
  MV_REQUIRE(row <= (1L << 30), "rows of %d heads of %d channels are too long", s.heads, s.dim);
  const int kept = s.dim - 2 * s.pairs, unit = kept % 8 == 0 ? 8 : kept % 4 == 0 ? 4 : kept % 2 == 0 ? 2 : 1;
  const int pieces = ((neighbours ? 2 : 1) * s.pairs + 7) / 8;
  Rotary k{s, 0, 0, pieces, kept / unit, unit, unit * dtype_size(dtype) <= 16 && kept / unit <= pieces ? kept / unit : 0, Divisor(std::max(1, s.pairs)), Divisor(std::max(1, pieces)), Divisor(s.heads), Divisor(std::max(1, kept / unit))};
  // Up to 4096 elements a workgroup (2 x 32768 x 8 heads of 64 in bf16: 37 us, with 8192 47, with 2048 44), fewer where that would leave compute
  // units without one
  const long spread = static_cast<long>(s.batch) * s.rows / 1024;
  k.block_rows = static_cast<int>(std::max(1L, std::min({4096L / row, 64L, kTable / std::max(1L, static_cast<long>(s.pairs)), static_cast<long>(s.rows), spread})));
  k.row_blocks = (s.rows + k.block_rows - 1) / k.block_rows;
  const long blocks = static_cast<long>(s.batch) * k.row_blocks;
  MV_REQUIRE(blocks < (1L << 31), "too many rows: %d in a batch of %d", s.rows, s.batch);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const size_t lds = sizeof(float2) * k.block_rows * s.pairs;
  MV_FLOATS(dtype, {
    const auto kernel = neighbours ? rotary<T, true> : rotary<T, false>;
    kernel<<<linear_grid(blocks, kThreads), kThreads, lds, st>>>(static_cast<const T *>(x), places, place_dtype, static_cast<const double *>(frequencies),
                                                                static_cast<T *>(y), k, back != 0);
  })
  return check_launch("rotary_positions");
}

// What the forward and backward kernels of cross attention share: tiles of keys and values (or of queries and gradients) in
// LDS, and products of 32 x 32 on the matrix cores.
//
// A product's second operand always stays in registers with one query (or key) per lane; its first one comes from a tile in
// LDS.  Results of a first product have the layout that the second operand of the next one wants (a lane keeps its column,
// its 16 rows are the second product's sum index in an order that the first operand follows), so that weights never leave
// the registers.
#pragma once
#include "rows.hpp"

namespace mv {

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kMostDim = 128;
constexpr float kLog2e = 1.44269504088896f;
// Scores beyond this (in powers of two) have their row's largest one taken off before they are scaled.  Otherwise scaling and
// the difference are one instruction, which rounds the largest one's product by up to 2^-24 of it: 2^-14 here, less than the
// weights' rounding to 16 bits; from 2^24 on whole powers of two, with which weights of 2^15 overflow float16.
constexpr float kFar = 1024.f;

struct AttentionArgs {
  const void *q, *k, *v;
  const unsigned char *mask;
  const int *lengths;
  int batch, queries, keys, heads, key_heads, dim;
  long qs[3], ks[3], vs[3], mask_stride;
  float scale;   // of the results; its magnitude times log2(e) scales the products, its sign goes into the queries
  __device__ __forceinline__ int length(int b) const { return lengths ? min(max(lengths[b], 0), keys) : keys; }
  __device__ __forceinline__ bool counts(int b, int j) const { return !mask || mask[b * mask_stride + j]; }
  // of the logarithms [batch, heads, queries], for a row of the output [batch, queries, heads]
  __device__ __forceinline__ long log_at(long row) const {
    const long i = row / heads, b = i / queries;
    return (b * heads + (row - i * heads)) * queries + (i - b * queries);
  }
  // (not zero: a key that does not count has a score of minus infinity, which has to stay that)
  __device__ __forceinline__ float factor() const {
    const float f = fabsf(scale) * kLog2e;
    return f == 0.f ? 1.17549435e-38f : f;
  }
};

// Rows of a head of keys: the heads that share it, query after query (neighbours in memory).
struct RowOf {
  int head, query;
  __device__ __forceinline__ RowOf(const AttentionArgs &a, int g, int row) : head(g), query(row) {
    if (a.heads != a.key_heads) {
      const unsigned group = a.heads / a.key_heads;
      query = static_cast<unsigned>(row) / group;
      head = g * group + (row - query * group);
    }
  }
};

// A workgroup's place.  Neighbours share what they read: tiles of the same keys where those are the longer side, heads of the
// same queries (of which two or four lie in a cache line) otherwise.
struct Place {
  int tile, split, g, b;
  bool in;
  __device__ __forceinline__ Place(const AttentionArgs &a, int tiles, int splits) {
    const unsigned all = static_cast<unsigned>(tiles) * splits * a.batch * a.key_heads;
    unsigned id = linear_block();
    in = id < all;
    if (!in) return;
    id = xcd_contiguous(id, all);
    const unsigned inner = a.queries > a.keys ? a.key_heads : tiles, outer = a.queries > a.keys ? tiles : a.key_heads;
    unsigned rest = id / inner;
    const int in_inner = id - rest * inner;
    split = 0;
    if (splits > 1) {
      split = rest % splits;
      rest /= splits;
    }
    b = rest / outer;
    const int in_outer = rest - b * outer;
    g = a.queries > a.keys ? in_inner : in_outer;
    tile = a.queries > a.keys ? in_outer : in_inner;
  }
};
// The share of `all` steps that a split does
__device__ __forceinline__ int share(int all, int split, int splits) {
  return splits == 1 ? (split ? all : 0) : static_cast<int>(static_cast<long>(all) * split / splits);
}

// ---- products of 32 x 32 ---------------------------------------------------------------------------------
// Row r of a result: lane % 32 is its column, register i holds row 8 (i / 4) + 4 (lane / 32) + i % 4.
__device__ __forceinline__ constexpr int result_row(int i, int half) { return 8 * (i / 4) + 4 * half + i % 4; }

template <typename T> struct Mma;
template <> struct Mma<__half> {
  typedef _Float16 piece __attribute__((ext_vector_type(8)));   // 8 of the 16 terms of a sum
  static __device__ __forceinline__ f32x16 mul(const piece &a, const piece &b, const f32x16 &c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ piece pack(const float *v) {
    piece r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = static_cast<_Float16>(v[i]);
    return r;
  }
};
template <> struct Mma<__hip_bfloat16> {
  typedef __bf16 piece __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x16 mul(const piece &a, const piece &b, const f32x16 &c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ piece pack(const float *v) {
    typedef float f32x8 __attribute__((ext_vector_type(8)));
    return __builtin_convertvector((f32x8{v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]}), piece);
  }
};

// ---- widths ----
// Kernels work on heads of W = 32, 64, 96 or 128 channels (zeros beyond the real ones); a tile's rows are powers of two.
constexpr int stored(int w) { return w == 96 ? 128 : w; }

// ---- tiles in LDS -------------------------------------------------------------------------------------------
// `Rows` rows of DP elements in pieces of 16 bytes.  Pieces of a row are exchanged by its number: eight rows of one column of
// pieces lie in different banks (whole rows are read so), and so do four rows of one pair of pieces (transposed ones).
template <typename T, int DP, int Rows> struct Tile {
  static constexpr int kPer = 16 / sizeof(T), kPieces = DP / kPer, kCount = Rows * kPieces;
  u32x4 at[kCount];
  static __device__ __forceinline__ int place(int row, int piece) {
    if constexpr (kPieces == 4) return row * 4 + (piece ^ ((row & 2) | ((row >> 2) & 1)));
    else return row * kPieces + (piece ^ ((row & 3) << 1 | ((row >> 2) & 1)));
  }
};

// The last piece of a row whose elements do not fill it: 16 bytes up to the row's end, moved down by the `over` elements that
// stand in front of the piece, with zeros behind.  One load and a few instructions: 2 x 1000 queries over 6912 keys, 4 heads of
// 100 channels, bf16: forward 52 us, dq 93, dk and dv 143 (an element at a time 100, 197 and 263).
template <typename T> __device__ __forceinline__ u32x4 moved_down(u32x4 r, int over) {
  const int bits = over * 8 * static_cast<int>(sizeof(T));   // 16 .. 112
  const unsigned long long low = r[0] | static_cast<unsigned long long>(r[1]) << 32, high = r[2] | static_cast<unsigned long long>(r[3]) << 32;
  const unsigned long long down = bits < 64 ? low >> bits | high << (64 - bits) : high >> (bits - 64), rest = bits < 64 ? high >> bits : 0;
  return u32x4{static_cast<unsigned>(down), static_cast<unsigned>(down >> 32), static_cast<unsigned>(rest), static_cast<unsigned>(rest >> 32)};
}

// 16 bytes of a row from element d < dim on, zeros beyond dim.  Ends: a piece that the row does not fill is read so; Raw: left to
// be moved down.  Otherwise it is read an element at a time.
template <typename T, bool Ends = true, bool Raw = false> __device__ __forceinline__ u32x4 load_piece(const T *row, int d, int dim) {
  constexpr int kPer = 16 / sizeof(T);
  if constexpr (Ends) {
    if (dim >= kPer) {
      const u32x4 r = reinterpret_cast<const Loose<u32x4, sizeof(T)> *>(row + min(d, dim - kPer))->v;
      return Raw || d + kPer <= dim ? r : moved_down<T>(r, d + kPer - dim);
    }
  } else if (d + kPer <= dim) {
    return reinterpret_cast<const Loose<u32x4, sizeof(T)> *>(row + d)->v;
  }
  u32x4 r = {0, 0, 0, 0};
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < 7; ++i)
      if (d + i < dim) r[i / 2] |= static_cast<unsigned>(reinterpret_cast<const unsigned short *>(row)[d + i]) << (i % 2 * 16);
  } else {
#pragma unroll
    for (int i = 0; i < 3; ++i)
      if (d + i < dim) r[i] = reinterpret_cast<const unsigned *>(row)[d + i];
  }
  return r;
}

// Two tiles of the same rows (keys and values, queries and gradients) on their way into LDS: each of 256 threads has one
// column of pieces, and every kStep-th row of it.
template <typename T, int DP, int Rows, bool Ends = true> struct Pair {
  using L = Tile<T, DP, Rows>;
  static constexpr int kStep = 256 / L::kPieces, kMine = Rows / kStep;
  static_assert(Rows % kStep == 0, "");
  u32x4 a[kMine], b[kMine];
  int row, d, dim;
  long stride_a, stride_b, at_a, at_b;   // of this thread's first piece
  int per = 1;   // heads of a query that follow each other
  long head_a = 0, head_b = 0;
  __device__ __forceinline__ Pair(long stride_a, long stride_b, int dim)
      : row(threadIdx.x / L::kPieces), d(threadIdx.x % L::kPieces * L::kPer), dim(dim), stride_a(stride_a), stride_b(stride_b) {
    const int from = first_element();
    at_a = row * stride_a + from, at_b = row * stride_b + from;
  }
  __device__ __forceinline__ int first_element() const { return Ends ? max(0, min(d, dim - L::kPer)) : d < dim ? d : 0; }
  // rows that are `inner` heads (a divisor of Rows) of each of Rows / inner queries
  __device__ __forceinline__ void heads(int inner, long head_a, long head_b) {
    per = inner;
    const int from = first_element();
    at_a = row_at(0, stride_a, head_a) + from, at_b = row_at(0, stride_b, head_b) + from;
    this->head_a = head_a, this->head_b = head_b;
  }
  __device__ __forceinline__ long row_at(int n, long stride, long head) const {
    const int r = row + n * kStep;
    if (per == 1) return r * stride;
    const int query = static_cast<unsigned>(r) / static_cast<unsigned>(per);
    return query * stride + (r - query * per) * head;
  }
  // Rows 0 .. left - 1 from two addresses on.  Whole tiles without a branch; what stands for elements that do not exist is
  // any value, to be replaced by put().
  __device__ __forceinline__ void load(const T *from_a, const T *from_b, int left) {
    if (left >= Rows && (Ends ? dim >= L::kPer : dim % L::kPer == 0) && kStep % per == 0) {
#pragma unroll
      for (int n = 0; n < kMine; ++n) {
        a[n] = reinterpret_cast<const Loose<u32x4, sizeof(T)> *>(from_a + n * (kStep / per) * stride_a + at_a)->v;
        b[n] = reinterpret_cast<const Loose<u32x4, sizeof(T)> *>(from_b + n * (kStep / per) * stride_b + at_b)->v;
      }
      return;
    }
#pragma unroll
    for (int n = 0; n < kMine; ++n) {
      a[n] = b[n] = u32x4{0, 0, 0, 0};
      if (row + n * kStep < left && d < dim) {
        a[n] = load_piece<T, Ends, Ends>(from_a + row_at(n, stride_a, head_a), d, dim);
        b[n] = load_piece<T, Ends, Ends>(from_b + row_at(n, stride_b, head_b), d, dim);
      }
    }
  }
  // zeros in the rows that a mask leaves out (they may hold anything, and NaN times a weight of zero is NaN)
  __device__ __forceinline__ void keep(const unsigned char *mask, int left) {
    bool use[kMine];
#pragma unroll
    for (int n = 0; n < kMine; ++n) use[n] = mask[min(row + n * kStep, left - 1)];
#pragma unroll
    for (int n = 0; n < kMine; ++n) {
      a[n] = use[n] ? a[n] : u32x4{0, 0, 0, 0};
      b[n] = use[n] ? b[n] : u32x4{0, 0, 0, 0};
    }
  }
  __device__ __forceinline__ void put(L (&to)[2]) {
    if (dim < DP && d >= dim) {
#pragma unroll
      for (int n = 0; n < kMine; ++n) a[n] = b[n] = u32x4{0, 0, 0, 0};
    }
    if (Ends && dim % L::kPer && dim >= L::kPer) {
      if (d < dim && d + L::kPer > dim) {
        const int over = L::kPer - dim % L::kPer;
#pragma unroll
        for (int n = 0; n < kMine; ++n) a[n] = moved_down<T>(a[n], over), b[n] = moved_down<T>(b[n], over);
      }
    }
#pragma unroll
    for (int n = 0; n < kMine; ++n) {
      const int at = L::place(row + n * kStep, d / L::kPer);
      to[0].at[at] = a[n], to[1].at[at] = b[n];
    }
  }
};

// Keys (or rows) that a workgroup has in LDS at a time, and whether twice: the next ones are written while these are read.
constexpr int staged_rows(int bytes, int dp, bool few, bool room) {
  return !few && !room ? 32 : few || (bytes == 2 && dp == 32) ? 128 : bytes == 4 && dp == 128 ? 32 : 64;
}
template <typename T, int DP, bool Few, bool Room = true> struct Staging {
  static constexpr int kRows = staged_rows(sizeof(T), DP, Few, Room);
  static constexpr int kBytes = 2 * kRows * DP * static_cast<int>(sizeof(T));
  static constexpr int kBuffers = kBytes <= 32768 ? 2 : 1;
};

// Whether the kernels for few rows or keys take this type and width: float32 heads of more than 64 channels would not fit
// into the registers.
template <typename T, int W> constexpr bool kHasFew = sizeof(T) == 2 || W <= 64;
inline bool has_few(int dtype, int dim) { return dtype != MV_F32 || dim <= 64; }

// What the backward pass takes from a score, `base` before scaling and `log` after it: the logarithm of the row's sum in one
// part, or the largest score first (float32: always, weights are then good to their last bits).  The difference is taken from the
// product as it was rounded in the forward pass too: a product that started from -most would not round it.
template <typename T> struct RowLog {
  float rest = -INFINITY, most = 0.f;   // (rows that do not exist are like those without a key)
  __device__ __forceinline__ void load(const AttentionArgs &a, const float *lse, long at) {
    rest = lse[at], most = lse[static_cast<long>(a.batch) * a.heads * a.queries + at];
  }
  __device__ __forceinline__ bool far(float factor) const { return sizeof(T) == 4 || fabsf(most) * factor > kFar; }
  __device__ __forceinline__ float base(float factor) const { return far(factor) ? most : 0.f; }
  __device__ __forceinline__ float log(float factor) const {
    return rest == -INFINITY ? INFINITY : far(factor) ? rest : fmaf(most, factor, rest);   // (weights of zero where no key counts)
  }
};

// v where bit `row` of the word is set, `other` where not (a field and a merge: two instructions in the forward pass; for
// `other` zero the compiler makes an and, a comparison and a selection of them)
__device__ __forceinline__ float where_bit(unsigned word, int row, float v, float other) {
  const unsigned all = static_cast<unsigned>(__builtin_amdgcn_sbfe(static_cast<int>(word), row, 1));
  return __uint_as_float((all & __float_as_uint(v)) | (~all & __float_as_uint(other)));
}

// Which of 64 keys count: bits for lanes' keys
__device__ __forceinline__ unsigned long long use_bits(const AttentionArgs &a, int b, int first, int count, int length) {
  const int lane = threadIdx.x & 63, j = first + lane;
  return __ballot(lane < count && j < length && a.counts(b, j));
}

// One column (a query, a key) per lane % 32, all W elements: the second operand of products over the elements.
template <typename T, int W, bool Ends = true> struct Column {
  static constexpr int kPer = 16 / sizeof(T), kCount = W / kPer / 2;
  u32x4 r[kCount];   // piece 2 n + lane / 32
  __device__ __forceinline__ void load(const T *row, bool use, int dim, int half) {
#pragma unroll
    for (int n = 0; n < kCount; ++n) {
      const int d = (2 * n + half) * kPer;
      r[n] = u32x4{0, 0, 0, 0};
      if (use && d < dim) r[n] = load_piece<T, Ends>(row, d, dim);
    }
  }
  __device__ __forceinline__ float dot(const Column &with) const {
    float sum = 0.f;
#pragma unroll
    for (int n = 0; n < kCount; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const unsigned x = r[n][i], y = with.r[n][i];
        if constexpr (sizeof(T) == 4) {
          sum = fmaf(__uint_as_float(x), __uint_as_float(y), sum);
        } else {
          sum = fmaf(Bits<T>::up(static_cast<unsigned short>(x & 0xffffu)), Bits<T>::up(static_cast<unsigned short>(y & 0xffffu)), sum);
          sum = fmaf(Bits<T>::up(static_cast<unsigned short>(x >> 16)), Bits<T>::up(static_cast<unsigned short>(y >> 16)), sum);
        }
      }
    return sum;
  }
  __device__ __forceinline__ void negate() {
#pragma unroll
    for (int n = 0; n < kCount; ++n) r[n] ^= sizeof(T) == 2 ? 0x80008000u : 0x80000000u;
  }
};

// 32 rows of a tile times the columns: over the elements of a row
template <typename T, int W, bool Ends, int DP, int Rows>
__device__ __forceinline__ f32x16 times(const Tile<T, DP, Rows> &tile, int first_row, const Column<T, W, Ends> &c, int lane) {
  f32x16 s = {};
  const int row = first_row + (lane & 31), half = lane >> 5;
#pragma unroll
  for (int n = 0; n < Column<T, W>::kCount; ++n) {
    const u32x4 a = tile.at[Tile<T, DP, Rows>::place(row, 2 * n + half)];
    if constexpr (sizeof(T) == 2) {
      using P = typename Mma<T>::piece;
      s = Mma<T>::mul(__builtin_bit_cast(P, a), __builtin_bit_cast(P, c.r[n]), s);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        s = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[i]), __uint_as_float(c.r[n][i]), s, 0, 0, 0);
    }
  }
  return s;
}

// sum[t] += (32 rows of a tile)^T weights, elements 32 t .. 32 t + 31 by the weights' columns: over the rows.  `w` is a
// result of times() (or what was made of it).  16 bits: the transposing load gives a lane four rows of its element, in the
// order in which the weights stand.
// Fine: what rounding takes from the weights is multiplied too (a second product with the same first operand).
template <bool Fine = false, typename T, int Tiles, int DP, int Rows>
__device__ __forceinline__ void add_transposed(const Tile<T, DP, Rows> &tile, int first_row, const float (&w)[16], f32x16 (&sum)[Tiles],
                                               int lane) {
  using L = Tile<T, DP, Rows>;
  const int half = lane >> 5;
  if constexpr (sizeof(T) == 2) {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    using P = typename Mma<T>::piece;
    // of 16 lanes: lane i reads 8 bytes of row i / 4, elements 4 (i % 4) .. + 3, and gets element i of the four rows
    const int in16 = lane & 15, row = first_row + 4 * half + in16 / 4, d = 16 * (lane >> 4 & 1) + 4 * (in16 % 4);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const P b = Mma<T>::pack(w + 8 * s);
      P b_low = {};
      if constexpr (Fine) {
        float rest[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) rest[i] = w[8 * s + i] - static_cast<float>(b[i]);
        b_low = Mma<T>::pack(rest);
      }
#pragma unroll
      for (int t = 0; t < Tiles; ++t) {
        s16x4 part[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = row + 16 * s + 8 * e;
          const char *from = reinterpret_cast<const char *>(&tile.at[L::place(r, 4 * t + d / 8)]) + d % 8 * 2;
          part[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(from));
        }
        const s16x8 a = __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7);
        sum[t] = Mma<T>::mul(__builtin_bit_cast(P, a), b, sum[t]);
        if constexpr (Fine) sum[t] = Mma<T>::mul(__builtin_bit_cast(P, a), b_low, sum[t]);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int row = first_row + result_row(i, 0) + 4 * half;
#pragma unroll
      for (int t = 0; t < Tiles; ++t) {
        const int d = 32 * t + (lane & 31);
        const float a = reinterpret_cast<const float *>(&tile.at[L::place(row, d / 4)])[d % 4];
        sum[t] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, w[i], sum[t], 0, 0, 0);
      }
    }
  }
}

// Sums of parts, in their order: `Slices` threads share the parts of one element of the first `count` (or of the second ones,
// which lie `splits` times `count` behind and go to `second`).
template <typename T, int Slices>
__global__ __launch_bounds__(256) void add_parts(const float *part, T *out, T *second, long count, int splits) {
  constexpr int kWide = 256 / Slices;
  __shared__ float sums[Slices][kWide];
  const int in = threadIdx.x % kWide, slice = threadIdx.x / kWide;
  long at = static_cast<long>(linear_block()) * kWide + in;
  const bool live = at < (second ? 2 : 1) * count, other = at >= count;
  if (other) at += (splits - 1) * count;   // (the first part of the second ones)
  float sum = 0.f;
  if (live) {
#pragma unroll 8
    for (int s = slice; s < splits; s += Slices) sum += part[s * count + at];
  }
  if constexpr (Slices > 1) {
    sums[slice][in] = sum;
    __syncthreads();
    if (slice) return;
#pragma unroll
    for (int i = 1; i < Slices; ++i) sum += sums[i][in];
  }
  if (!live) return;
  if (other) second[at - splits * count] = store_cast<T>(sum);
  else out[at] = store_cast<T>(sum);
}

// The other half of the wavefront has the other rows of the same column.
__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32); }

// What rounding to T takes away from v (nothing where v is not finite)
template <typename T> __device__ __forceinline__ float rest_of(float v) {
  if constexpr (sizeof(T) == 4) return 0.f;
  const T r = store_cast<T>(v);
  const float rest = v - mv::load(&r);
  return rest == rest ? rest : 0.f;
}

// Four neighbouring elements of a row of `dim` elements
template <typename T> __device__ __forceinline__ void store_quad(T *row, int d, int dim, float a, float b, float c, float e) {
  const float v[4] = {a, b, c, e};
  if (d + 4 <= dim) {
    if constexpr (sizeof(T) == 2) {
      const u32x2 r = {pack2<T>(a, b), pack2<T>(c, e)};
      reinterpret_cast<Loose<u32x2, 2> *>(row + d)->v = r;
    } else {
      reinterpret_cast<Loose<f32x4, 4> *>(row + d)->v = f32x4{a, b, c, e};
    }
  } else {
#pragma unroll
    for (int i = 0; i < 3; ++i)
      if (d + i < dim) row[d + i] = store_cast<T>(v[i]);
  }
}

// 32 elements of a column's results (as product results stand) to a row from element `first` on.  16 bits: the halves of the
// wavefront exchange what they have, so that each lane writes eight neighbours.
template <typename T> __device__ __forceinline__ void store_results(T *row, int first, int dim, int half, const float (&v)[16]) {
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      unsigned w[2][2];   // [register group 2 a + .][pair]
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) w[i][e] = pack2<T>(v[4 * (2 * a + i) + 2 * e], v[4 * (2 * a + i) + 2 * e + 1]);
      u32x4 r;   // lower half: elements 16 a .. + 7, upper half: 16 a + 8 .. + 15
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const auto both = __builtin_amdgcn_permlane32_swap(w[0][e], w[1][e], false, false);
        r[e] = both[0], r[2 + e] = both[1];
      }
      const int d = first + 16 * a + 8 * half;
      if (d + 8 <= dim) {
        reinterpret_cast<Loose<u32x4, 2> *>(row + d)->v = r;
      } else {
#pragma unroll
        for (int i = 0; i < 7; ++i)
          if (d + i < dim) reinterpret_cast<unsigned short *>(row)[d + i] = static_cast<unsigned short>(r[i / 2] >> (i % 2 * 16));
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) store_quad(row, first + 8 * i + 4 * half, dim, v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
  }
}

// The same for a head of `dim` channels, for the plans: no more splits than there are tiles.  `few` and `room` as the kernels give
// them to Staging.
inline int tile_rows(int dtype, int dim, bool few, bool room = true) {
  return staged_rows(dtype == MV_F32 ? 4 : 2, stored(dim <= 32 ? 32 : dim <= 64 ? 64 : dim <= 96 ? 96 : 128), few, room);
}
inline long parts_of(long count, long each) { return (count + each - 1) / each; }

inline int attention_sizes(const mv_attention_shape *s, int dtype) {
  MV_REQUIRE(s, "the shape is missing");
  MV_REQUIRE(dtype == MV_F32 || dtype == MV_F16 || dtype == MV_BF16, "dtype %d is not float32, float16 or bfloat16", dtype);
  MV_REQUIRE(s->batch >= 0 && s->queries >= 0 && s->keys >= 0, "wrong sizes: batch %d, %d queries, %d keys", s->batch, s->queries, s->keys);
  MV_REQUIRE(s->key_heads > 0 && s->heads > 0 && s->heads % s->key_heads == 0, "%d heads cannot share %d heads of keys", s->heads, s->key_heads);
  // (workgroups and rows of a head of keys are counted in 32 bits)
  const long most = (1L << 31) - 256, heads = static_cast<long>(s->batch) * s->key_heads, rows = static_cast<long>(s->heads / s->key_heads) * s->queries;
  MV_REQUIRE(rows < most && s->keys < most && heads * (rows / 128 + 1) < most && heads * (s->keys / 128 + 1) < most, "too many heads, queries or keys");
  MV_REQUIRE(s->dim > 0 && s->dim <= kMostDim, "heads of %d channels: 1 to %d are possible", s->dim, kMostDim);
  return MV_OK;
}

inline AttentionArgs attention_arguments(const mv_attention_shape *s, const void *q, const void *k, const void *v, const void *mask, const void *lengths, float scale) {
  AttentionArgs a{q, k, v, static_cast<const unsigned char *>(mask), static_cast<const int *>(lengths), s->batch, s->queries, s->keys,
                  s->heads, s->key_heads, s->dim, {}, {}, {}, static_cast<long>(s->mask_stride), scale};
  for (int i = 0; i < 3; ++i) a.qs[i] = s->q_strides[i], a.ks[i] = s->k_strides[i], a.vs[i] = s->v_strides[i];
  return a;
}

}  // namespace mv

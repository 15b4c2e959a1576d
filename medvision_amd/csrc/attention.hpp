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

struct AttentionArgs {
  const void *q, *k, *v;
  const unsigned char *mask;
  const int *lengths;
  int batch, queries, keys, heads, key_heads, dim;
  long qs[3], ks[3], vs[3], mask_stride;
  float scale;   // of the results; its magnitude times log2(e) scales the products, its sign goes into the queries
  __device__ __forceinline__ int length(int b) const { return lengths ? min(max(lengths[b], 0), keys) : keys; }
  __device__ __forceinline__ bool counts(int b, int j) const { return !mask || mask[b * mask_stride + j]; }
  __device__ __forceinline__ float factor() const { return fabsf(scale) * kLog2e; }
};

// Rows of a head of keys: the queries of all heads that share it, one after the other.
struct RowOf {
  int head, query;
  __device__ __forceinline__ RowOf(const AttentionArgs &a, int g, int row) : head(g * (a.heads / a.key_heads) + row / a.queries), query(row % a.queries) {}
};

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

// ---- tiles in LDS -------------------------------------------------------------------------------------------
// `Rows` rows of DP elements in pieces of 16 bytes.  Pieces of a row are exchanged by its number, so that eight rows of one
// column of pieces lie in different banks.
template <typename T, int DP, int Rows> struct Tile {
  static constexpr int kPer = 16 / sizeof(T), kPieces = DP / kPer, kCount = Rows * kPieces;
  u32x4 at[kCount];
  static __device__ __forceinline__ int place(int row, int piece) {
    if constexpr (kPieces == 4) return row * 4 + (piece ^ ((row >> 1) & 3));
    else return row * kPieces + (piece ^ (row & 7));
  }
};

// 16 bytes of a row from element d on, zeros beyond dim
template <typename T> __device__ __forceinline__ u32x4 load_piece(const T *row, int d, int dim) {
  constexpr int kPer = 16 / sizeof(T);
  if (d + kPer <= dim) return reinterpret_cast<const Loose<u32x4, sizeof(T)> *>(row + d)->v;
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

// What a thread of `Threads` brings of a tile: loaded ahead into registers, put into LDS later.
template <typename T, int DP, int Rows, int Threads> struct Carry {
  using L = Tile<T, DP, Rows>;
  static constexpr int kMine = (L::kCount + Threads - 1) / Threads;
  u32x4 r[kMine];
  // rows `first` + 0 .. Rows - 1 of those below `last`; `row(i)` gives the address of one, `use(i)` whether it counts
  template <typename Row, typename Use>
  __device__ __forceinline__ void load(int thread, int first, int last, int dim, const Row &row, const Use &use) {
#pragma unroll
    for (int n = 0; n < kMine; ++n) {
      const int at = thread + n * Threads, i = first + at / L::kPieces, d = at % L::kPieces * L::kPer;
      r[n] = u32x4{0, 0, 0, 0};
      if (i < last && d < dim && use(i)) r[n] = load_piece<T>(row(i), d, dim);
    }
  }
  __device__ __forceinline__ void put(int thread, L &to) const {
#pragma unroll
    for (int n = 0; n < kMine; ++n) {
      const int at = thread + n * Threads;
      if (L::kCount % Threads == 0 || at < L::kCount) to.at[L::place(at / L::kPieces, at % L::kPieces)] = r[n];
    }
  }
};

// One column (a query, a key) per lane % 32, all DP elements: the second operand of products over the elements.
template <typename T, int DP> struct Column {
  static constexpr int kPer = 16 / sizeof(T), kCount = DP / kPer / 2;
  u32x4 r[kCount];   // piece 2 n + lane / 32
  __device__ __forceinline__ void load(const T *row, bool use, int dim, int half) {
#pragma unroll
    for (int n = 0; n < kCount; ++n) {
      const int d = (2 * n + half) * kPer;
      r[n] = u32x4{0, 0, 0, 0};
      if (use && d < dim) r[n] = load_piece<T>(row, d, dim);
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
template <typename T, int DP, int Rows>
__device__ __forceinline__ f32x16 times(const Tile<T, DP, Rows> &tile, int first_row, const Column<T, DP> &c, int lane) {
  f32x16 s = {};
  const int row = first_row + (lane & 31), half = lane >> 5;
#pragma unroll
  for (int n = 0; n < Column<T, DP>::kCount; ++n) {
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
template <typename T, int DP, int Rows>
__device__ __forceinline__ void add_transposed(const Tile<T, DP, Rows> &tile, int first_row, const float (&w)[16], f32x16 (&sum)[DP / 32],
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
#pragma unroll
      for (int t = 0; t < DP / 32; ++t) {
        s16x4 part[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = row + 16 * s + 8 * e;
          const char *from = reinterpret_cast<const char *>(&tile.at[L::place(r, 4 * t + d / 8)]) + d % 8 * 2;
          part[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(from));
        }
        const s16x8 a = __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7);
        sum[t] = Mma<T>::mul(__builtin_bit_cast(P, a), b, sum[t]);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int row = first_row + result_row(i, 0) + 4 * half;
#pragma unroll
      for (int t = 0; t < DP / 32; ++t) {
        const int d = 32 * t + (lane & 31);
        const float a = reinterpret_cast<const float *>(&tile.at[L::place(row, d / 4)])[d % 4];
        sum[t] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, w[i], sum[t], 0, 0, 0);
      }
    }
  }
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

// Product of 16-bit rows with weights in 4 bits (e2m1) and a scale for each group of 32, 64 or 128 columns of a row:
//   y[m, n] = sum over groups g of  s[n, g] sum_k x[m, k] w[n, k]  + bias[n]
//
// The values of 4-bit codes (0, 1/2, 1, 3/2, 2, 3, 4, 6 and their negatives) are exact in 16 bits, and so are the matrix
// units' products; a group's sum is scaled in 32 bits when it is added.
//
// The weights of a row are blocks of 128 columns, 64 bytes.  The four bytes of eight neighbouring columns stay together
// (two codes a byte, the first one in its low half); piece 4 s + g of a block's sixteen stands at place 4 g + s.  One
// 16-byte load then brings lane group g its columns of four products of 32 columns, each within one group of a scale.
#include "parts.hpp"
#include "rows.hpp"

#include <algorithm>
#include <type_traits>

namespace mv {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// Eight codes to 16 bits, two by two; their products with eight columns of 16 rows, added to `sum`
template <typename T> struct Matrix;
template <> struct Matrix<__half> {
  static __device__ __forceinline__ u32x4 values(unsigned codes) {
    return {__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, 1.f, 0)),
            __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, 1.f, 1)),
            __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, 1.f, 2)),
            __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, 1.f, 3))};
  }
  static __device__ __forceinline__ f32x4 product(const u32x4 &a, const u32x4 &b, const f32x4 &sum) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), sum, 0, 0, 0);
  }
};
template <> struct Matrix<__hip_bfloat16> {
  static __device__ __forceinline__ u32x4 values(unsigned codes) {
    return {__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, 1.f, 0)),
            __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, 1.f, 1)),
            __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, 1.f, 2)),
            __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, 1.f, 3))};
  }
  static __device__ __forceinline__ f32x4 product(const u32x4 &a, const u32x4 &b, const f32x4 &sum) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), sum, 0, 0, 0);
  }
};

// Eight columns of a row as they are, zeros from `left` on
template <typename T> __device__ __forceinline__ u32x4 columns8(const T *p, int left) {
  if (left >= 8) return reinterpret_cast<const Loose<u32x4, 2> *>(p)->v;
  u32x4 r = {0u, 0u, 0u, 0u};
  if (left <= 0) return r;
  unsigned v[7];
#pragma unroll
  for (int i = 0; i < 7; ++i) v[i] = reinterpret_cast<const unsigned short *>(p)[min(i, left - 1)];
#pragma unroll
  for (int i = 0; i < 7; ++i) r[i / 2] |= i < left ? v[i] << (i % 2 * 16) : 0u;
  return r;
}

template <typename T> struct Product {
  const T *x;
  const unsigned char *w;
  const float *scales;
  const T *bias;
  T *y;
  float *part;   // [splits, rows, outputs], NULL: y
  long rows;
  long stride;   // of x's rows, in elements
  int inputs, outputs, blocks, m_tiles, n_tiles, splits;
};

// ---- tiles ---------------------------------------------------------------------------------------------------------
// A workgroup takes 128 rows and 128 outputs, each of its 2 x 2 wavefronts 64 x 64 of them.  Rows and weights of a block of 128
// columns go through LDS, without registers on the way (x: rows in whole pieces of 16 bytes), the next block's while this one is
// multiplied; scales go to the lanes that want them.  A row of x is 256 bytes there, sixteen pieces, piece c of row r at c ^ (r & 15); a row of
// weights four, piece g at g ^ turned(r): reads of 16 rows side by side spread over all banks.
// 4000 x 4096 x 4096 in bf16 with groups of 128, 64, 32: 130, 147, 172 us = 1.03, 0.91, 0.78 PFLOP/s (a plain product of the library: 1.21;
// this kernel without its scales: 1.17); 2000 x 12544 x 1024 with groups of 64 60 us and 7 for the join.  No one thing bounds it: of the first
// 128 us its matrix instructions alone take 70, with the additions of scaled sums (an instruction for each result and group) 80, with reads
// of LDS 95, its loads alone 68.  Two workgroups share a compute unit, so that one multiplies while the other waits for its operands:
// tiles of 128 x 256, of which one fits, took 145 us, and two teams of wavefronts in one workgroup, which join in LDS, 172.  Without gain:
// products of 32 x 32, matrix instructions with the additions of the group before in between, scales brought a block ahead, two blocks
// under way at once.
constexpr int kTile = 128, kTileThreads = 256, kTileRows = kTile * 256, kStage = kTileRows + kTile * 64;   // bytes of the rows, of a block
__device__ __forceinline__ int turned(int row) { return (row / 2 & 3) ^ (row / 8 & 1); }

template <typename T, int Group> __global__ __launch_bounds__(kTileThreads, 2) void product_tiles4(const Product<T> k) {
  constexpr int kScales = kBlock / Group;
  __shared__ __attribute__((aligned(16))) unsigned char lds[2 * kStage];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r16 = lane & 15, g = lane >> 4;
  const int wm = wave % 2, wn = wave / 2;
  // tiles in an order in which neighbouring workgroups of a die share rows and weights: four rows of tiles at a time, for rows are four
  // times as many bytes as weights (1000 x 12544 x 1024: 44 us, of eight 50)
  const int tiles = k.m_tiles * k.n_tiles;
  unsigned id = linear_block();
  if (id >= static_cast<unsigned>(tiles) * k.splits) return;
  const int split = id / tiles;
  id = xcd_contiguous(id % tiles, tiles);
  const int band = id / (4 * k.n_tiles), in_band = id % (4 * k.n_tiles), tall = min(4, k.m_tiles - 4 * band);
  const long m0 = (4L * band + in_band % tall) * kTile;
  const int n0 = in_band / tall * kTile;
  const int first = static_cast<int>(static_cast<long>(k.blocks) * split / k.splits), last = static_cast<int>(static_cast<long>(k.blocks) * (split + 1) / k.splits);

  // What a thread brings of a block: pieces of 16 bytes, in the order in which they stand in LDS
  constexpr int kPiecesX = kTile * 16 / kTileThreads, kPiecesW = kTile * 4 / kTileThreads;
  static_assert(kTile * 16 % kTileThreads == 0 && kTile * 4 % kTileThreads == 0, "");
  const T *x_from[kPiecesX];
  int x_column[kPiecesX];
  const unsigned char *w_from[kPiecesW];
#pragma unroll
  for (int i = 0; i < kPiecesX; ++i) {
    const int at = i * kTileThreads + threadIdx.x, row = at / 16;
    x_column[i] = ((at % 16) ^ (row & 15)) * 8;
    x_from[i] = k.x + min(m0 + row, k.rows - 1) * k.stride + x_column[i];
  }
#pragma unroll
  for (int i = 0; i < kPiecesW; ++i) {
    const int at = i * kTileThreads + threadIdx.x, row = at / 4;
    w_from[i] = k.w + static_cast<long>(min(n0 + row, k.outputs - 1)) * k.blocks * 64 + ((at % 4) ^ turned(row)) * 16;
  }
  const float *s_from[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) s_from[u] = k.scales + static_cast<long>(min(n0 + wn * 64 + u * 16 + r16, k.outputs - 1)) * k.blocks * kScales;

  float scale[4][kScales];
  auto bring = [&](int b) {
    unsigned char *const to = lds + (b & 1) * kStage + wave * 1024;
#pragma unroll
    for (int i = 0; i < kPiecesX; ++i) {   // (of a piece behind the row's end: the row's first one, which zeros take the place of)
      const T *const from = b * kBlock + x_column[i] < k.inputs ? x_from[i] + b * kBlock : x_from[i] - x_column[i];
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)from,
                                       (__attribute__((address_space(3))) void *)(to + i * kTileThreads * 16), 16, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < kPiecesW; ++i)
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)(w_from[i] + b * 64L),
                                       (__attribute__((address_space(3))) void *)(to + kTileRows + i * kTileThreads * 16), 16, 0, 0);
  };
  f32x4 acc[4][4] = {};
  bring(first);
  for (int b = first; b < last; ++b) {
    __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0): what this wavefront brought has arrived (a barrier alone does not promise that)
    __syncthreads();   // this block's operands are there, and nobody reads the place of the next ones
    unsigned char *const here = lds + (b & 1) * kStage;
    if ((b + 1) * kBlock > k.inputs) {   // the columns behind the rows' ends
#pragma unroll
      for (int i = 0; i < kPiecesX; ++i)
        if (b * kBlock + x_column[i] >= k.inputs) *reinterpret_cast<u32x4 *>(here + (i * kTileThreads + threadIdx.x) * 16) = u32x4{0u, 0u, 0u, 0u};
      __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int i = 0; i < kScales; ++i) scale[u][i] = s_from[u][b * kScales + i];
    if (b + 1 < last) bring(b + 1);
    u32x4 x[4][4], w[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int row = wn * 64 + u * 16 + r16;
      w[u] = *reinterpret_cast<const u32x4 *>(here + kTileRows + row * 64 + (g ^ turned(row)) * 16);
    }
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = wm * 64 + t * 16 + r16;
        x[t][i] = *reinterpret_cast<const u32x4 *>(here + row * 256 + ((4 * i + g) ^ (row & 15)) * 16);
      }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      f32x4 d[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const u32x4 v = Matrix<T>::values(w[u][i]);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          if (i % (Group / 32) == 0) d[t] = f32x4{0.f, 0.f, 0.f, 0.f};
          d[t] = Matrix<T>::product(x[t][i], v, d[t]);
        }
        if ((i + 1) % (Group / 32) == 0) {
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[t][u][j] = fmaf(d[t][j], scale[u][i / (Group / 32)], acc[t][u][j]);
        }
      }
    }
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int n = n0 + wn * 64 + u * 16 + r16;
    if (n >= k.outputs) continue;
    const float add = k.bias && !k.part ? load(k.bias + n) : 0.f;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const long m = m0 + wm * 64 + t * 16 + 4 * g + j;
        if (m >= k.rows) continue;
        if (k.part) k.part[(split * k.rows + m) * k.outputs + n] = acc[t][u][j];
        else k.y[m * k.outputs + n] = store_cast<T>(acc[t][u][j] + add);
      }
  }
}

// ---- a row or two ------------------------------------------------------------------------------------------------------
// Bound by reading the weights once, in vector instructions (a matrix instruction would have fifteen rows of nothing): a wavefront
// has four outputs and sixteen blocks of them at a time, 1024 neighbouring bytes of each; a lane has a quarter of a block, the columns
// 32 s + 8 g .. + 7 of lane group g.  `along` wavefronts of a workgroup share the blocks and join in LDS.  Codes go to 32 bits (two in an
// instruction), so that small float16 values count in full.  One row of 87808 x 1024 in bf16 with groups of 128: 11.5 us (48 MB, 4.2 TB/s);
// sixteen rows' form takes 16 with its join, and 4096 x 4096 9.3 instead of 5.0 us (two rows: 9 and 6.3).
// A wavefront whose row of weights has no more than half its blocks takes other outputs beside them (Sides): one row of 1024 x 87808 with
// groups of 64 13.7 us, without 23.5, of 256 x 87808 5.4 and 23.
constexpr int kDotOutputs = 4, kDotBlocks = 16, kMostAlong = 8, kMostSides = 8;

template <typename T, int M, int Group, int Sides> __global__ __launch_bounds__(64 * kMostAlong) void product_dots(const Product<T> k, int along) {
  constexpr int kScales = kBlock / Group, kWidth = 64 / Sides, kSpan = kDotBlocks / Sides, kWide = kDotOutputs * Sides;
  __shared__ float part[kMostAlong][M][kDotOutputs * Sides];
  unsigned id = linear_block();
  if (id >= static_cast<unsigned>(k.n_tiles) * k.splits) return;
  const int split = id / k.n_tiles, waves = blockDim.x >> 6;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane & 3, side = lane / kWidth, in = lane % kWidth >> 2;
  const int n0 = ((id - split * k.n_tiles) * (waves / along) + wave / along) * kWide;
  const int chunks = (k.blocks + kSpan - 1) / kSpan;
  const int first = static_cast<int>(static_cast<long>(chunks) * split / k.splits) + wave % along, last = static_cast<int>(static_cast<long>(chunks) * (split + 1) / k.splits);
  const unsigned char *w_at[kDotOutputs];
  const float *s_at[kDotOutputs];
#pragma unroll
  for (int u = 0; u < kDotOutputs; ++u) {
    const long n = min(n0 + side * kDotOutputs + u, k.outputs - 1);
    w_at[u] = k.w + n * k.blocks * 64 + g * 16;
    s_at[u] = k.scales + n * k.blocks * kScales;
  }
  struct Operands {
    u32x4 w[kDotOutputs], x[M][4];
    float s[kDotOutputs][kScales];
  };
  auto bring = [&](Operands &o, int chunk) {
    const int at = chunk * kSpan + in, b = min(at, k.blocks - 1);   // (behind the last one: that one, times zero)
#pragma unroll
    for (int u = 0; u < kDotOutputs; ++u) {
      o.w[u] = *reinterpret_cast<const u32x4 *>(w_at[u] + b * 64L);
#pragma unroll
      for (int i = 0; i < kScales; ++i) o.s[u][i] = s_at[u][static_cast<long>(b) * kScales + i];
    }
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = b * kBlock + i * 32 + g * 8;
        o.x[m][i] = columns8(k.x + m * k.stride + c, at < k.blocks ? k.inputs - c : 0);
      }
  };
  float acc[M][kDotOutputs] = {};
  Operands next;
  if (first < last) bring(next, first);
  for (int chunk = first; chunk < last; chunk += along) {
    const Operands o = next;
    if (chunk + along < last) bring(next, chunk + along);
    const bool there = chunk * kSpan + in < k.blocks;
    float sum[M][kDotOutputs] = {};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float x[M][8];
#pragma unroll
      for (int m = 0; m < M; ++m)
#pragma unroll
        for (int j = 0; j < 8; ++j) x[m][j] = Bits<T>::up(static_cast<unsigned short>(o.x[m][i][j / 2] >> (j % 2 * 16)));
#pragma unroll
      for (int u = 0; u < kDotOutputs; ++u) {
        const f32x2 v[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(o.w[u][i], 1.f, 0), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(o.w[u][i], 1.f, 1),
                            __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(o.w[u][i], 1.f, 2), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(o.w[u][i], 1.f, 3)};
#pragma unroll
        for (int m = 0; m < M; ++m) {
#pragma unroll
          for (int j = 0; j < 8; ++j) sum[m][u] = fmaf(x[m][j], v[j / 2][j % 2], sum[m][u]);
          if ((i + 1) % (Group / 32) == 0) {
            acc[m][u] = there ? fmaf(sum[m][u], o.s[u][i / (Group / 32)], acc[m][u]) : acc[m][u];
            sum[m][u] = 0.f;
          }
        }
      }
    }
  }
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int u = 0; u < kDotOutputs; ++u) {
#pragma unroll
      for (int d = kWidth / 2; d; d >>= 1) acc[m][u] += __shfl_xor(acc[m][u], d);
      if (lane % kWidth == 0) part[wave][m][side * kDotOutputs + u] = acc[m][u];
    }
  __syncthreads();
  if (wave % along || lane >= M * kWide) return;
  const int m = lane / kWide, n = n0 + lane % kWide;
  float y = 0.f;
  for (int i = 0; i < along; ++i) y += part[wave + i][m][lane % kWide];
  if (n >= k.outputs) return;
  if (k.part) k.part[(split * k.rows + m) * k.outputs + n] = y;
  else k.y[m * k.outputs + n] = store_cast<T>(k.bias ? y + load(k.bias + n) : y);
}

// ---- few rows -------------------------------------------------------------------------------------------------------
// 16 TN outputs and 16 TM rows, straight from memory into the operands' registers.  `Along` wavefronts (all of a workgroup's, or two)
// take turns at the blocks of their share of the sum and join in LDS.  Bound by memory, and by loads of rows that every workgroup repeats:
// 13 rows of 8100 x 8190 in float16 with groups of 32 13.4 us (42 MB, 3.1 TB/s); with four wavefronts 16.0, with four tiles of outputs 16.6.
// From 17 rows on four wavefronts with four tiles: 32 x 4096 x 4096 with groups of 64 11.6 us (with eight
// 15.3, eight of two tiles 12.1), 64 x 12544 x 1024 17.7.
constexpr int waves_of(int tm) { return tm <= 1 ? 8 : 4; }
constexpr int tiles_wide(int tm) { return tm <= 1 ? 2 : 4; }

template <typename T, int TM, int Group, int Along>
__global__ __launch_bounds__(64 * waves_of(TM), 2) void product_rows4(const Product<T> k) {
  constexpr int TN = tiles_wide(TM), kScales = kBlock / Group, kWaves = waves_of(TM);
  __shared__ f32x4 part[kWaves - 1][TN * TM][64];
  unsigned id = linear_block();
  if (id >= static_cast<unsigned>(k.m_tiles) * k.n_tiles * k.splits) return;
  const int n_tile = id % k.n_tiles;
  id /= k.n_tiles;
  const int split = id % k.splits;
  const long m0 = static_cast<long>(id / k.splits) * 16 * TM;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r16 = lane & 15, g = lane >> 4;
  const int own = wave % Along, n0 = (n_tile * (kWaves / Along) + wave / Along) * 16 * TN;   // (its place among those that share the blocks)
  const int first = static_cast<int>(static_cast<long>(k.blocks) * split / k.splits), last = static_cast<int>(static_cast<long>(k.blocks) * (split + 1) / k.splits);
  const T *x_at[TM];
  const unsigned char *w_at[TN];
  const float *s_at[TN];
#pragma unroll
  for (int t = 0; t < TM; ++t) x_at[t] = k.x + min(m0 + t * 16 + r16, k.rows - 1) * k.stride;
#pragma unroll
  for (int u = 0; u < TN; ++u) {
    const long n = min(n0 + u * 16 + r16, k.outputs - 1);
    w_at[u] = k.w + n * k.blocks * 64 + g * 16;
    s_at[u] = k.scales + n * k.blocks * kScales;
  }
  struct Operands {
    u32x4 w[TN], x[TM][4];
    float s[TN][kScales];
  };
  auto bring_weights = [&](Operands &o, int b) {
#pragma unroll
    for (int u = 0; u < TN; ++u) {
      o.w[u] = *reinterpret_cast<const u32x4 *>(w_at[u] + b * 64L);
#pragma unroll
      for (int i = 0; i < kScales; ++i) o.s[u][i] = s_at[u][static_cast<long>(b) * kScales + i];
    }
  };
  auto bring_rows = [&](Operands &o, int b, auto whole) {
#pragma unroll
    for (int t = 0; t < TM; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = b * kBlock + i * 32 + g * 8;
        if constexpr (whole) o.x[t][i] = reinterpret_cast<const Loose<u32x4, 2> *>(x_at[t] + c)->v;
        else o.x[t][i] = columns8(x_at[t] + c, k.inputs - c);
      }
  };
  f32x4 acc[TM][TN] = {};
  auto multiply = [&](const Operands &o) {
#pragma unroll
    for (int u = 0; u < TN; ++u) {
      f32x4 d[TM];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const u32x4 v = Matrix<T>::values(o.w[u][i]);
#pragma unroll
        for (int t = 0; t < TM; ++t) {
          if (i % (Group / 32) == 0) d[t] = f32x4{0.f, 0.f, 0.f, 0.f};
          d[t] = Matrix<T>::product(o.x[t][i], v, d[t]);
          if ((i + 1) % (Group / 32) == 0) {
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[t][u][j] = fmaf(d[t][j], o.s[u][i / (Group / 32)], acc[t][u][j]);
          }
        }
      }
    }
  };
  // Whole blocks with nothing to ask on the way, so that another one is under way whole while one is multiplied (where there are
  // registers for that: else the next one's weights); then the one that ends with the rows.  20 x 8100 x 8190 with groups of 32: 19 us, where each
  // load asks whether the row is long enough 21.5; 13 rows 13.4 and 13.8.
  const int whole = min(last, k.inputs / kBlock), mine = max(0, (whole - first - own + Along - 1) / Along), b0 = first + own;
  const std::true_type all;
  int n = 0;
  if constexpr (TM == 1 || (TM == 2 && Group > 32)) {
    auto bring = [&](Operands &o, int n) { bring_weights(o, b0 + n * Along), bring_rows(o, b0 + n * Along, all), __builtin_amdgcn_sched_barrier(0); };   // (stays where it is)
    Operands one, two;
    if (mine > 1) {
      bring(one, 0);
      bring(two, 1);
      for (; n + 3 < mine; n += 2) {
        multiply(one);
        bring(one, n + 2);
        multiply(two);
        bring(two, n + 3);
      }
      multiply(one);   // (two or three are left)
      if (n + 2 < mine) bring(one, n + 2);
      multiply(two);
      if (n + 2 < mine) multiply(one);
    } else if (mine == 1) {
      bring(one, 0);
      multiply(one);
    }
  } else {
    Operands next;
    if (mine > 0) bring_weights(next, b0);
    for (; n < mine; ++n) {
      Operands o = next;
      bring_rows(o, b0 + n * Along, all);
      if (n + 1 < mine) bring_weights(next, b0 + (n + 1) * Along);
      multiply(o);
    }
  }
  if (whole < last && (whole - first) % Along == own) {
    Operands o;
    bring_weights(o, whole);
    bring_rows(o, whole, std::false_type());
    multiply(o);
  }
  if (own) {
#pragma unroll
    for (int u = 0; u < TN; ++u)
#pragma unroll
      for (int t = 0; t < TM; ++t) part[wave - 1][u * TM + t][lane] = acc[t][u];
  }
  __syncthreads();
  if (own) return;
#pragma unroll
  for (int u = 0; u < TN; ++u) {
    const int n = n0 + u * 16 + r16;
    if (n >= k.outputs) continue;
    const float add = k.bias && !k.part ? load(k.bias + n) : 0.f;
#pragma unroll
    for (int t = 0; t < TM; ++t) {
#pragma unroll
      for (int i = 0; i < Along - 1; ++i) acc[t][u] += part[wave + i][u * TM + t][lane];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const long m = m0 + t * 16 + 4 * g + j;
        if (m >= k.rows) continue;
        if (k.part) k.part[(split * k.rows + m) * k.outputs + n] = acc[t][u][j];
        else k.y[m * k.outputs + n] = store_cast<T>(acc[t][u][j] + add);
      }
    }
  }
}

// ---- weights to 4 bits ------------------------------------------------------------------------------------------
// A thread has eight neighbouring columns; those of a group are neighbouring lanes.
template <typename T>
__global__ __launch_bounds__(256) void quantize_groups(const T *w, unsigned *q, float *scales, long pieces, int columns, int blocks, int group) {
  const long at = static_cast<long>(linear_block()) * 256 + threadIdx.x;
  if (at >= pieces) return;   // (whole blocks of sixteen lanes)
  const int o = static_cast<int>(at & 15);
  const long block = at >> 4, row = block / blocks;
  const int c = static_cast<int>(block - row * blocks) * kBlock + o * 8;
  float v[8], most = 0.f;
  load8(w + row * columns + c, columns - c, v);
#pragma unroll
  for (int i = 0; i < 8; ++i) most = max_abs(most, v[i]);
  for (int d = 1; d < group / 8; d *= 2) most = max_abs(most, __shfl_xor(most, d));
  const float s = most / 6.f, scale = s < kLeastScale ? kLeastScale : s, inverse = 1.f / scale;   // (NaN stays)
  unsigned codes = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {   // to the nearest level, halves to the even code
    const float t = v[i] * inverse, a = fabsf(t);
    const unsigned code = (a > 0.25f) + (a >= 0.75f) + (a > 1.25f) + (a >= 1.75f) + (a > 2.5f) + (a >= 3.5f) + (a > 5.f);
    codes |= (code + (t < 0.f ? 8u : 0u)) << (4 * i);
  }
  q[block * 16 + (o & 3) * 4 + (o >> 2)] = codes;
  if (o % (group / 8) == 0) scales[at / (group / 8)] = scale;
}

// ---- which kernel --------------------------------------------------------------------------------------------------
enum Kind { kDots, kFew1, kFew2, kFew4, kTiles };
struct Plan {
  int kind, m_tiles, n_tiles, splits;
  int along = 1, waves = 4, sides = 1;   // of kDots; of kFew the first two
};

constexpr int kDotRows = 2;
int ceil_div(long a, long b) { return static_cast<int>((a + b - 1) / b); }

// The form by the number of rows (figures beside the kernels), splits of the sum until there is work for every compute unit: a split
// costs the parts' way through memory (and a launch, 3 - 4 us), so that each has two turns of its wavefronts at least (a row or two: one, of
// sixteen blocks), in tiles four blocks (100 x 4096 x 4096: 22 us, with eight 24.5).
Plan plan_of(long rows, int blocks, int outputs) {
  if (rows <= kDotRows) {
    const int chunks = ceil_div(blocks, kDotBlocks);
    int along = 1, sides = 1;
    while (along < kMostAlong && along < chunks) along *= 2;
    // (as many outputs side by side as leave a thousand workgroups: 1024 x 16384 4.9 us, without 5.9, of 8192 outputs 4.9 both ways)
    while (sides < kMostSides && 2 * sides * blocks <= kDotBlocks && outputs >= 1024L * 4 * kDotOutputs * sides) sides *= 2;
    const int waves = std::max(4, along), n = ceil_div(outputs, waves / along * kDotOutputs * sides);
    return {kDots, 1, n, std::max(1, std::min(chunks / along, 256 / n)), along, waves, sides};
  }
  if (rows <= 64) {
    const int kind = rows <= 16 ? kFew1 : rows <= 32 ? kFew2 : kFew4, tm = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
    // (two wavefronts on few blocks while there is a workgroup for every compute unit: 13 x 256 x 50000 5.8 us, all eight 9.1, 13 x 1024 x 50000 16
    // and 18.2; 13 x 2048 x 50000 28.4 and 26.9)
    const int waves = waves_of(tm), along = blocks <= 8 && outputs >= 256L * 16 * tiles_wide(tm) * (waves / 2) ? 2 : waves;
    const int n = ceil_div(outputs, 16 * tiles_wide(tm) * (waves / along));
    return {kind, 1, n, std::max(1, std::min(blocks / (2 * waves), 256 * 8 / waves / n)), along, waves};
  }
  const int m = ceil_div(rows, 128), n = ceil_div(outputs, 128);
  return {kTiles, m, n, static_cast<int>(std::max(1L, std::min(blocks / 4L, 512 / (static_cast<long>(m) * n))))};
}

template <typename T, int Group, int Sides> void dots(const Plan &p, const Product<T> &k, long groups, hipStream_t s) {
  if (k.rows == 1) product_dots<T, 1, Group, Sides><<<linear_grid(groups, 64 * p.waves), 64 * p.waves, 0, s>>>(k, p.along);
  else product_dots<T, 2, Group, Sides><<<linear_grid(groups, 64 * p.waves), 64 * p.waves, 0, s>>>(k, p.along);
}

template <typename T, int TM, int Group> void few(const Plan &p, const Product<T> &k, long groups, hipStream_t s) {
  constexpr int kWaves = waves_of(TM);
  if (p.along == kWaves) product_rows4<T, TM, Group, kWaves><<<linear_grid(groups, 64 * kWaves), 64 * kWaves, 0, s>>>(k);
  else product_rows4<T, TM, Group, 2><<<linear_grid(groups, 64 * kWaves), 64 * kWaves, 0, s>>>(k);
}

template <typename T, int Group> void launch(const Plan &p, const Product<T> &k, hipStream_t s) {
  const long groups = static_cast<long>(p.m_tiles) * p.n_tiles * p.splits;
  switch (p.kind) {
    case kDots:
      if (p.sides == 1) dots<T, Group, 1>(p, k, groups, s);
      else if (p.sides == 2) dots<T, Group, 2>(p, k, groups, s);
      else if (p.sides == 4) dots<T, Group, 4>(p, k, groups, s);
      else dots<T, Group, 8>(p, k, groups, s);
      break;
    case kFew1: few<T, 1, Group>(p, k, groups, s); break;
    case kFew2: few<T, 2, Group>(p, k, groups, s); break;
    case kFew4: few<T, 4, Group>(p, k, groups, s); break;
    default: product_tiles4<T, Group><<<linear_grid(groups, 256), 256, 0, s>>>(k);
  }
}

// Rows as tiles read them: with zeros up to whole blocks, 16-byte aligned.  A thread has eight columns.
template <typename T> __global__ __launch_bounds__(256) void pad_rows(const T *x, u32x4 *to, long pieces, int inputs, int blocks) {
  const long at = static_cast<long>(linear_block()) * 256 + threadIdx.x;
  if (at >= pieces) return;
  const long row = at / (blocks * 16L);
  const int c = static_cast<int>(at - row * (blocks * 16L)) * 8;
  to[at] = columns8(x + row * inputs + min(c, inputs - 1), inputs - c);
}
size_t padded_bytes(long rows, int blocks) { return static_cast<size_t>(rows) * blocks * kBlock * 2; }
size_t part_bytes(const Plan &p, long rows, int outputs) { return p.splits > 1 ? sizeof(float) * p.splits * static_cast<size_t>(rows) * outputs : 0; }

template <typename T>
int product(const void *x, const void *w, const void *scales, const void *bias, void *y, long rows, int inputs, int outputs, int group,
            void *workspace, size_t workspace_bytes, hipStream_t s) {
  const int blocks = ceil_div(inputs, kBlock);
  Plan p = plan_of(rows, blocks, outputs);
  // Rows that tiles cannot read are copied first; where there is no room for that, they go straight to registers.
  const bool tiles = p.kind == kTiles, odd = tiles && (inputs % 8 || reinterpret_cast<uintptr_t>(x) % 16);
  const size_t pad = odd ? padded_bytes(rows, blocks) : 0;
  if (!workspace) workspace_bytes = 0;
  const bool pads = odd && pad <= workspace_bytes && reinterpret_cast<uintptr_t>(workspace) % 16 == 0;
  if (odd && !pads) p = {kFew4, ceil_div(rows, 64), ceil_div(outputs, 16 * tiles_wide(4)), 1, waves_of(4), waves_of(4)};
  const size_t at = pads ? pad : 0;
  if (workspace_bytes - at < part_bytes(p, rows, outputs)) p.splits = 1;
  Product<T> k{static_cast<const T *>(x), static_cast<const unsigned char *>(w), static_cast<const float *>(scales), static_cast<const T *>(bias),
               static_cast<T *>(y), p.splits > 1 ? reinterpret_cast<float *>(static_cast<char *>(workspace) + at) : nullptr, rows, inputs, inputs, outputs, blocks,
               p.m_tiles, p.n_tiles, p.splits};
  if (pads) {
    const long pieces = rows * blocks * 16;
    pad_rows<<<linear_grid((pieces + 255) / 256, 256), 256, 0, s>>>(k.x, static_cast<u32x4 *>(workspace), pieces, inputs, blocks);
    k.x = static_cast<const T *>(workspace), k.stride = static_cast<long>(blocks) * kBlock, k.inputs = blocks * kBlock;
  }
  if (group == 32) launch<T, 32>(p, k, s);
  else if (group == 64) launch<T, 64>(p, k, s);
  else launch<T, 128>(p, k, s);
  if (k.part) launch_join(k.part, k.bias, k.y, rows * outputs, outputs, p.splits, s);
  return check_launch("group_linear");
}

}  // namespace
}  // namespace mv

using namespace mv;

extern "C" {

int mv_quantize_groups(const void *weight, void *q, void *scales, int64_t rows, int columns, int group, int dtype, void *stream) {
  MV_REQUIRE(group == 32 || group == 64 || group == 128, "groups of %d columns: 32, 64 or 128 are possible", group);
  MV_REQUIRE(rows >= 0 && rows < (1L << 31) && columns > 0 && columns <= (1 << 30), "wrong sizes: %ld rows of %d columns", static_cast<long>(rows), columns);
  if (rows == 0) return MV_OK;
  MV_REQUIRE(weight && q && scales, "a tensor is missing");
  const int blocks = ceil_div(columns, kBlock);
  const long pieces = rows * blocks * 16;
  MV_FLOATS(dtype, {
    quantize_groups<T><<<linear_grid((pieces + 255) / 256, 256), 256, 0, static_cast<hipStream_t>(stream)>>>(
        static_cast<const T *>(weight), static_cast<unsigned *>(q), static_cast<float *>(scales), pieces, columns, blocks, group);
  })
  return check_launch("quantize_groups");
}

size_t mv_group_linear_workspace_bytes(int64_t rows, int inputs, int outputs) {
  if (rows <= 0 || inputs <= 0 || outputs <= 0) return 0;
  const int blocks = ceil_div(inputs, kBlock);
  const Plan p = plan_of(rows, blocks, outputs);
  return part_bytes(p, rows, outputs) + (p.kind == kTiles && inputs % 8 ? padded_bytes(rows, blocks) : 0);
}

int mv_group_linear(const void *x, const void *weight, const void *scales, const void *bias, void *y, int64_t rows, int inputs, int outputs,
                    int group, int dtype, void *workspace, size_t workspace_bytes, void *stream) {
  MV_REQUIRE(dtype == MV_F16 || dtype == MV_BF16, "dtype %d is not float16 or bfloat16", dtype);
  MV_REQUIRE(group == 32 || group == 64 || group == 128, "groups of %d columns: 32, 64 or 128 are possible", group);
  MV_REQUIRE(rows >= 0 && rows < (1L << 31) - 256 && inputs > 0 && inputs <= (1 << 30) && outputs >= 0 && outputs < (1L << 31) - 256,
             "wrong sizes: %ld rows, %d inputs, %d outputs", static_cast<long>(rows), inputs, outputs);
  if (rows == 0 || outputs == 0) return MV_OK;
  MV_REQUIRE(x && weight && scales && y, "a tensor is missing");
  MV_REQUIRE(reinterpret_cast<uintptr_t>(weight) % 16 == 0, "the weight has to be 16-byte aligned");
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return dtype == MV_F16 ? product<__half>(x, weight, scales, bias, y, rows, inputs, outputs, group, workspace, workspace_bytes, s)
                         : product<__hip_bfloat16>(x, weight, scales, bias, y, rows, inputs, outputs, group, workspace, workspace_bytes, s);
}

}  // extern "C"

// Product of 8-bit floats (e4m3) with a scale for each row and 128 columns of the activations and for each 128 x 128 block
// of the weights:  y[m, n] = sum over blocks b of  sx[m, b] sw[n / 128, b] sum_k qx[m, 128 b + k] qw[n, 128 b + k]  + bias[n]
//
// One v_mfma 16x16x128 takes a whole block of 128: it starts from zero, and its result is added to the sum in 32 bits with
// the two scales' product.  The weights are its first operand, so that a lane's results lie in one row of y (one scale per
// tile and lane, four neighbouring results).
#include "rows.hpp"

#include <algorithm>

namespace mv {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f32x4 block_product(const i32x8 &w, const i32x8 &x) {
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  // (scales of 0: the instruction without scales)
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, zero, 0, 0, 0, 0, 0, 0);
}

__device__ __forceinline__ i32x8 join(const i32x4 &a, const i32x4 &b) { return {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]}; }

// Where results go: y itself, or a part of the sums in 32 bits.
template <typename T> struct Results {
  T *y;
  const T *bias;
  float *part;   // [splits, rows, outputs], NULL: y
  long rows;
  int outputs;
};

// Results of TN tiles along row m, four neighbours of every 16 from n on
template <typename T, int TN> __device__ __forceinline__ void store_row(const Results<T> &to, int split, long m, int n, const f32x4 (&v)[TN]) {
  if (m >= to.rows) return;
  if (to.part) {
    float *const at = to.part + (split * to.rows + m) * to.outputs;
#pragma unroll
    for (int u = 0; u < TN; ++u) {
      const int c = n + 16 * u;
      if (c + 4 <= to.outputs) reinterpret_cast<Loose<f32x4, 4> *>(at + c)->v = v[u];
      else
#pragma unroll
        for (int i = 0; i < 3; ++i)
          if (c + i < to.outputs) at[c + i] = v[u][i];
    }
    return;
  }
  T *const at = to.y + m * to.outputs;
#pragma unroll
  for (int u = 0; u < TN; ++u) {
    const int c = n + 16 * u;
    f32x4 r = v[u];
    if (to.bias) {
#pragma unroll
      for (int i = 0; i < 4; ++i) r[i] += load(to.bias + min(c + i, to.outputs - 1));
    }
    const u32x2 bits = {pack2<T>(r[0], r[1]), pack2<T>(r[2], r[3])};
    if (c + 4 <= to.outputs) reinterpret_cast<Loose<u32x2, 2> *>(at + c)->v = bits;
    else
#pragma unroll
      for (int i = 0; i < 3; ++i)
        if (c + i < to.outputs) reinterpret_cast<unsigned short *>(at)[c + i] = static_cast<unsigned short>(bits[i / 2] >> (i % 2 * 16));
  }
}

// ---- tiles ----------------------------------------------------------------------------------------------
// A workgroup takes BM rows and BN outputs; WM x WN wavefronts share the tile, WK groups of them take every WK-th block of
// the sum.  Both operands go from memory to LDS without registers (16 bytes per lane, the next blocks while these are
// multiplied).  A row of a block is 128 bytes, eight pieces of 16; piece c of row r stands at c ^ (r & 7), so that the 16
// rows of an operand that one instruction reads spread over all banks (no conflicts).
//
// 256 x 256 with eight wavefronts of 64 x 128: 16384 x 4096 x 4096 253 - 261 us = 2.1 - 2.2 PFLOP/s (a plain product of the
// library: 2.34), 8192^3 479 us = 2.30 (the same inputs each time).  Matrix units 46 % busy, vector units 37 % (the additions of the
// scaled products to the sums), LDS reads 21 %; they overlap less than whole, and every fourth step the five wavefronts that put scales
// into LDS wait for the next block first (a store to LDS behind loads into LDS).
// 128 x 128 with twice four wavefronts of 64 x 64, where there are fewer than 192 of the large tiles (4000 x 12544 x 1024:
// 68 - 72 us = 1.4 - 1.5 PFLOP/s; 160 with the large ones, 80 with those split in four): the loads alone take 52 us (803 MB from the
// L2s, 15.6 TB/s), reads and products 48, and both share the LDS; all wavefronts wait for the next blocks in every second step, for the
// scales' sake.  Matrix units and vector units 29 % busy each.
template <int BM, int BN, int WM, int WN, int WK> struct Tiles {
  static constexpr int kThreads = 64 * WM * WN * WK, kTM = BM / WM / 16, kTN = BN / WN / 16;
  static constexpr int kStage = (BM + BN) * kBlock;   // bytes of one block of both operands
  static constexpr int kLds = 2 * WK * kStage, kScales = BM + BN / kBlock;
};

template <typename T, int BM, int BN, int WM, int WN, int WK>
__global__ __launch_bounds__(64 * WM * WN * WK, WM *WN *WK / 4) void product_tiles(
    const unsigned char *q, const float *qs, const unsigned char *w, const float *ws, const Results<T> to, int rows, int inputs,
    int outputs, int m_tiles, int n_tiles, int splits) {
  using S = Tiles<BM, BN, WM, WN, WK>;
  __shared__ __attribute__((aligned(16))) unsigned char lds[S::kLds];
  __shared__ float scale[2][4][WK][S::kScales];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int group = wave / (WM * WN), in_group = wave % (WM * WN), wm = in_group % WM, wn = in_group / WM;
  // tiles in an order in which neighbouring workgroups of a die share rows and weights: eight rows of tiles at a time
  const int tiles = m_tiles * n_tiles;
  unsigned id = linear_block();
  if (id >= static_cast<unsigned>(tiles) * splits) return;
  const int split = id / tiles;
  id = xcd_contiguous(id % tiles, tiles);
  const int band = id / (8 * n_tiles), in_band = id % (8 * n_tiles), tall = min(8, m_tiles - 8 * band);
  const int m0 = (8 * band + in_band % tall) * BM, n0 = in_band / tall * BN;
  const int blocks = inputs / kBlock, first = static_cast<int>(static_cast<long>(blocks) * split / splits),
            last = static_cast<int>(static_cast<long>(blocks) * (split + 1) / splits), steps = (last - first + WK - 1) / WK;

  // What this wavefront brings: 8 rows (1024 bytes) per instruction.
  constexpr int kRows8 = (BM + BN) / 8, kMine = kRows8 / (WM * WN);
  static_assert(kRows8 % (WM * WN) == 0, "");
  const int lr = lane >> 3, piece = (lane & 7) ^ lr;
  const unsigned char *from[kMine];
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const int row = (in_group * kMine + i) * 8 + lr;   // of the stage: activations, then weights
    from[i] = (row < BM ? q + static_cast<long>(min(m0 + row, rows - 1)) * inputs
                        : w + static_cast<long>(min(n0 + row - BM, outputs - 1)) * inputs) + piece * 16;
  }
  auto bring = [&](int step) {
    const int b = min(first + step * WK + group, last - 1);
    unsigned char *to = lds + ((step & 1) * WK + group) * S::kStage + in_group * kMine * 1024;
#pragma unroll
    for (int i = 0; i < kMine; ++i)
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)(from[i] + static_cast<long>(b) * kBlock),
                                       (__attribute__((address_space(3))) void *)(to + i * 1024), 16, 0, 0);
  };

  const int r16 = lane & 15, g = lane >> 4;
  // The scales of four steps at a time, by one thread for a row (and one for 128 outputs), through LDS: read by every lane
  // that needs them they would be as many cache lines as the operands.
  const int mine = threadIdx.x % (64 * WM * WN);
  const bool brings_scales = mine < S::kScales;
  const float *const scale_at = mine < BM ? qs + static_cast<long>(min(m0 + mine, rows - 1)) * blocks
                                          : ws + static_cast<long>(min(n0 + (mine - BM) * kBlock, outputs - 1) / kBlock) * blocks;
  float ahead[4];
  auto bring_scales = [&](int step) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (brings_scales) ahead[i] = scale_at[min(first + (step + i) * WK + group, last - 1)];
  };
  auto put_scales = [&](int step) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (brings_scales) scale[(step >> 2) & 1][i][group][mine] = ahead[i];
  };

  f32x4 acc[S::kTM][S::kTN] = {};
  bring_scales(0);
  bring(0);
  put_scales(0);
  // The next weights are on their way while these are multiplied, and the last products are added meanwhile.  Where there are
  // registers for it, the last weights of a step are multiplied in the next one, while its first operands come from LDS
  // (4000 x 12544 x 1024: 72.4 us with, 73.6 without; tiles of 256 x 256 would spill 210 registers).
  constexpr bool kLater = S::kTM * S::kTN <= 16;
  i32x8 x0[S::kTM] = {}, x1[S::kTM] = {}, v = {};
  float scale_before[S::kTM] = {};
  const int p0 = (g ^ (r16 & 7)) * 16, p1 = ((g + 4) ^ (r16 & 7)) * 16;
  auto piece_of = [&](const unsigned char *tile, int row16) {
    // piece g and piece g + 4 of the row: any order of k serves, as long as both operands have the same
    const unsigned char *row = tile + (row16 * 16 + r16) * kBlock;
    return join(*reinterpret_cast<const i32x4 *>(row + p0), *reinterpret_cast<const i32x4 *>(row + p1));
  };
  auto add = [&](int u, const f32x4 (&d)[S::kTM], const float (&s)[S::kTM]) {
#pragma unroll
    for (int t = 0; t < S::kTM; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[t][u][i] = fmaf(d[t][i], s[t], acc[t][u][i]);
  };
  auto one_step = [&](int step, i32x8 (&now)[S::kTM], const i32x8 (&before)[S::kTM]) {
    __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0): what this wavefront brought has arrived (a barrier alone does not promise that)
    __syncthreads();   // this step's operands are there, and nobody reads the place of the next ones
    if ((step & 3) == 0) bring_scales(step + 4);
    if (step + 1 < steps) bring(step + 1);
    if ((step & 3) == 3) put_scales(step + 1);
    if (WK > 1 && first + step * WK + group >= last) {   // (the last step of a group that has no block left)
#pragma unroll
      for (int t = 0; t < S::kTM; ++t)
        if (kLater) now[t] = before[t];
      return;
    }
    const unsigned char *xs = lds + ((step & 1) * WK + group) * S::kStage, *wsm = xs + BM * kBlock;
    const float *const factors = scale[(step >> 2) & 1][step & 3][group];
    float s[S::kTM];
    i32x8 next = piece_of(wsm, wn * S::kTN);
#pragma unroll
    for (int t = 0; t < S::kTM; ++t) now[t] = piece_of(xs, wm * S::kTM + t);
#pragma unroll
    for (int t = 0; t < S::kTM; ++t) s[t] = factors[(wm * S::kTM + t) * 16 + r16] * factors[BM + wn * S::kTN * 16 / kBlock];
    __builtin_amdgcn_sched_barrier(0);
    f32x4 d[2][S::kTM];
    if constexpr (kLater) {
#pragma unroll
      for (int t = 0; t < S::kTM; ++t) d[1][t] = block_product(v, before[t]);
      __builtin_amdgcn_sched_barrier(0);
    }
    v = next;
    static_assert(S::kTN % 2 == 0, "");
#pragma unroll
    for (int u = 0; u < (kLater ? S::kTN - 1 : S::kTN); ++u) {
      if (u + 1 < S::kTN) next = piece_of(wsm, wn * S::kTN + u + 1);
#pragma unroll
      for (int t = 0; t < S::kTM; ++t) d[u & 1][t] = block_product(v, now[t]);
      if (u) add(u - 1, d[(u - 1) & 1], s);
      else if (kLater) add(S::kTN - 1, d[1], scale_before);
      v = next;
#pragma unroll
      for (int t = 0; t < S::kTM; ++t) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);   // a matrix instruction
        if (t == 0) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);   // LDS reads
        if (u || kLater) __builtin_amdgcn_sched_group_barrier(0x2, 4, 0);   // four additions
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (kLater) {
      add(S::kTN - 2, d[0], s);
#pragma unroll
      for (int t = 0; t < S::kTM; ++t) scale_before[t] = s[t];
    } else {
      add(S::kTN - 1, d[1], s);
    }
  };
  if constexpr (kLater) {
    for (int step = 0; step < steps; step += 2) {
      one_step(step, x0, x1);
      if (step + 1 < steps) one_step(step + 1, x1, x0);
    }
  } else {
    for (int step = 0; step < steps; ++step) one_step(step, x0, x0);
  }
  auto finish = [&](const i32x8 (&before)[S::kTM]) {
    f32x4 d[S::kTM];
#pragma unroll
    for (int t = 0; t < S::kTM; ++t) d[t] = block_product(v, before[t]);
    add(S::kTN - 1, d, scale_before);
  };
  if constexpr (kLater) {
    if (steps & 1) finish(x0);
    else finish(x1);
  }
  if (WK > 1) {   // the groups' sums, in their order
    f32x4 *const part = reinterpret_cast<f32x4 *>(lds);
    const int at = in_group * 64 + lane;
    for (int from_group = 1; from_group < WK; ++from_group) {
      __syncthreads();
      if (group == from_group) {
#pragma unroll
        for (int u = 0; u < S::kTN; ++u)
#pragma unroll
          for (int t = 0; t < S::kTM; ++t) part[(u * S::kTM + t) * (64 * WM * WN) + at] = acc[t][u];
      }
      __syncthreads();
      if (group == 0) {
#pragma unroll
        for (int u = 0; u < S::kTN; ++u)
#pragma unroll
          for (int t = 0; t < S::kTM; ++t) acc[t][u] += part[(u * S::kTM + t) * (64 * WM * WN) + at];
      }
    }
  }
  __syncthreads();   // the operands, and the groups' sums, have been read: their place is free
  if (group) return;
  // Whole tiles of results in 16 bits: through LDS, so that 256 (128) neighbouring bytes of a row are written at a time; as
  // they stand, 32 bytes of each of 16 rows.
  constexpr int kCols = S::kTN * 16, kUnits = kCols / 8;   // pieces of 16 bytes of a row of this wavefront
  const int m_first = m0 + wm * S::kTM * 16, n_first = n0 + wn * kCols;
  if (!to.part && m_first + S::kTM * 16 <= rows && n_first + kCols <= outputs && outputs % 8 == 0 && reinterpret_cast<unsigned long>(to.y) % 16 == 0) {
    unsigned char *const mine = lds + in_group * (S::kTM * 16 * kCols * 2);
    static_assert(WM * WN * S::kTM * 16 * kCols * 2 <= S::kLds, "");
#pragma unroll
    for (int u = 0; u < S::kTN; ++u) {
      float add[4] = {};
      if (to.bias) {
#pragma unroll
        for (int i = 0; i < 4; ++i) add[i] = load(to.bias + n_first + u * 16 + 4 * g + i);
      }
#pragma unroll
      for (int t = 0; t < S::kTM; ++t) {
        const f32x4 v = acc[t][u];
        const int row = t * 16 + r16, unit = (u * 2 + g / 2) ^ (row % kUnits);
        *reinterpret_cast<u32x2 *>(mine + (row * kUnits + unit) * 16 + g % 2 * 8) =
            u32x2{pack2<T>(v[0] + add[0], v[1] + add[1]), pack2<T>(v[2] + add[2], v[3] + add[3])};
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // (a wavefront reads only what it wrote)
#pragma unroll
    for (int i = 0; i < S::kTM * 16 * kUnits / 64; ++i) {
      const int at = i * 64 + lane, row = at / kUnits, unit = at % kUnits;
      *reinterpret_cast<u32x4 *>(to.y + static_cast<long>(m_first + row) * outputs + n_first + unit * 8) =
          *reinterpret_cast<const u32x4 *>(mine + (row * kUnits + (unit ^ (row % kUnits))) * 16);
    }
    return;
  }
#pragma unroll
  for (int t = 0; t < S::kTM; ++t) {
    store_row(to, split, m0 + (wm * S::kTM + t) * 16 + r16, n0 + wn * S::kTN * 16 + 4 * g, acc[t]);
  }
}

// ---- few rows -----------------------------------------------------------------------------------------------
// Bound by reading the weights once: 64 outputs and 16 TM rows per workgroup, straight from memory into the operands'
// registers, the next block's while this one is multiplied.  The four wavefronts take turns at the blocks of the
// workgroup's share of the sum and join in LDS.  8 x 87808 x 1024: 17 us and 3 us for the join of 32 splits (90 MB of
// weights: 4.5 TB/s in all).
template <typename T, int TM>
__global__ __launch_bounds__(256) void product_rows(const unsigned char *q, const float *qs, const unsigned char *w, const float *ws,
                                                    const Results<T> to, int rows, int inputs, int outputs, int m_tiles, int n_tiles,
                                                    int splits) {
  constexpr int TN = 4;
  __shared__ f32x4 part[3][TN * TM][64];
  unsigned id = linear_block();
  if (id >= static_cast<unsigned>(m_tiles) * n_tiles * splits) return;
  const int n_tile = id % n_tiles;
  id /= n_tiles;
  const int split = id % splits, m0 = id / splits * 16 * TM, n0 = n_tile * 16 * TN;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r16 = lane & 15, g = lane >> 4;
  const int blocks = inputs / kBlock, first = static_cast<int>(static_cast<long>(blocks) * split / splits),
            last = static_cast<int>(static_cast<long>(blocks) * (split + 1) / splits);
  const unsigned char *x_at[TM], *w_at[TN];
  const float *sx_at[TM];
#pragma unroll
  for (int t = 0; t < TM; ++t) {
    const long m = min(m0 + t * 16 + r16, rows - 1);
    x_at[t] = q + m * inputs + g * 16;
    sx_at[t] = qs + m * blocks;
  }
#pragma unroll
  for (int u = 0; u < TN; ++u) w_at[u] = w + static_cast<long>(min(n0 + u * 16 + r16, outputs - 1)) * inputs + g * 16;
  const float *sw_at = ws + static_cast<long>(n0 / kBlock) * blocks;

  i32x8 x[TM], v[TN];
  float s[TM];
  auto bring = [&](int b) {
    const long k = static_cast<long>(b) * kBlock;
#pragma unroll
    for (int u = 0; u < TN; ++u)
      v[u] = join(*reinterpret_cast<const i32x4 *>(w_at[u] + k), *reinterpret_cast<const i32x4 *>(w_at[u] + k + 64));
#pragma unroll
    for (int t = 0; t < TM; ++t)
      x[t] = join(*reinterpret_cast<const i32x4 *>(x_at[t] + k), *reinterpret_cast<const i32x4 *>(x_at[t] + k + 64));
#pragma unroll
    for (int t = 0; t < TM; ++t) s[t] = sx_at[t][b] * sw_at[b];
  };
  f32x4 acc[TM][TN] = {};
  if (first + wave < last) bring(first + wave);
  for (int b = first + wave; b < last; b += 4) {
    i32x8 x1[TM], v1[TN];
    float s1[TM];
#pragma unroll
    for (int t = 0; t < TM; ++t) x1[t] = x[t], s1[t] = s[t];
#pragma unroll
    for (int u = 0; u < TN; ++u) v1[u] = v[u];
    if (b + 4 < last) bring(b + 4);
#pragma unroll
    for (int u = 0; u < TN; ++u)
#pragma unroll
      for (int t = 0; t < TM; ++t) {
        const f32x4 d = block_product(v1[u], x1[t]);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[t][u][i] = fmaf(d[i], s1[t], acc[t][u][i]);
      }
  }
  if (wave) {
#pragma unroll
    for (int u = 0; u < TN; ++u)
#pragma unroll
      for (int t = 0; t < TM; ++t) part[wave - 1][u * TM + t][lane] = acc[t][u];
  }
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int u = 0; u < TN; ++u)
#pragma unroll
    for (int t = 0; t < TM; ++t) {
#pragma unroll
      for (int i = 0; i < 3; ++i) acc[t][u] += part[i][u * TM + t][lane];
    }
#pragma unroll
  for (int t = 0; t < TM; ++t) store_row(to, split, m0 + t * 16 + r16, n0 + 4 * g, acc[t]);
}

// The parts' sum, in a fixed order: `Slices` threads share the parts of a result.
template <typename T, int Slices>
__global__ __launch_bounds__(256) void join_parts(const float *part, const T *bias, T *y, long count, int outputs, int splits) {
  constexpr int kWide = 256 / Slices;
  __shared__ float sums[Slices][kWide];
  const int in = threadIdx.x % kWide, slice = threadIdx.x / kWide;
  const long at = static_cast<long>(linear_block()) * kWide + in;
  float sum = 0.f;
  if (at < count) {
#pragma unroll 4
    for (int s = slice; s < splits; s += Slices) sum += part[s * count + at];
  }
  if constexpr (Slices > 1) {
    sums[slice][in] = sum;
    __syncthreads();
    if (slice) return;
#pragma unroll
    for (int i = 1; i < Slices; ++i) sum += sums[i][in];
  }
  if (at >= count) return;
  if (bias) sum += load(bias + at % outputs);
  y[at] = store_cast<T>(sum);
}

// ---- which kernel --------------------------------------------------------------------------------------------
enum Kind { kFew1, kFew2, kFew4, kTile128, kTile256 };
struct Plan {
  int kind, m_tiles, n_tiles, splits;
};

int ceil_div(long a, long b) { return static_cast<int>((a + b - 1) / b); }

// Few rows up to 64 (64 x 12544 x 1024 14.6 us; of 128, which tiles take, 19.4).  Sums are split where there are fewer
// workgroups than compute units (512 for few rows), into shares of eight blocks at least; a split costs the parts' way through memory (4000 x 1024 x 4096 in one piece 25 us, in two 77), so
// that no more are made than fill the chip once (1000 x 4096 x 1024: 30.0 us in one piece, 21.0 in four, 30.7 in eight).
Plan plan_of(long rows, int inputs, int outputs) {
  const int blocks = inputs / kBlock;
  if (rows <= 64) {
    const int kind = rows <= 16 ? kFew1 : rows <= 32 ? kFew2 : kFew4;
    const int n_tiles = ceil_div(outputs, 64);
    return {kind, 1, n_tiles, std::max(1, std::min(blocks / 8, 512 / n_tiles))};
  }
  const long big = static_cast<long>(ceil_div(rows, 256)) * ceil_div(outputs, 256);
  if (big >= 192) return {kTile256, ceil_div(rows, 256), ceil_div(outputs, 256), 1};
  const int m = ceil_div(rows, 128), n = ceil_div(outputs, 128);
  return {kTile128, m, n, std::max(1, std::min(blocks / 8, 256 / (m * n)))};
}

template <typename T>
void launch(const Plan &p, const void *q, const void *qs, const void *w, const void *ws, const Results<T> &to, int rows, int inputs,
            int outputs, hipStream_t s) {
  const long groups = static_cast<long>(p.m_tiles) * p.n_tiles * p.splits;
  const auto *q8 = static_cast<const unsigned char *>(q), *w8 = static_cast<const unsigned char *>(w);
  const auto *qf = static_cast<const float *>(qs), *wf = static_cast<const float *>(ws);
  switch (p.kind) {
    case kFew1: product_rows<T, 1><<<linear_grid(groups, 256), 256, 0, s>>>(q8, qf, w8, wf, to, rows, inputs, outputs, p.m_tiles, p.n_tiles, p.splits); break;
    case kFew2: product_rows<T, 2><<<linear_grid(groups, 256), 256, 0, s>>>(q8, qf, w8, wf, to, rows, inputs, outputs, p.m_tiles, p.n_tiles, p.splits); break;
    case kFew4: product_rows<T, 4><<<linear_grid(groups, 256), 256, 0, s>>>(q8, qf, w8, wf, to, rows, inputs, outputs, p.m_tiles, p.n_tiles, p.splits); break;
    case kTile128: product_tiles<T, 128, 128, 2, 2, 2><<<linear_grid(groups, 512), 512, 0, s>>>(q8, qf, w8, wf, to, rows, inputs, outputs, p.m_tiles, p.n_tiles, p.splits); break;
    default: product_tiles<T, 256, 256, 4, 2, 1><<<linear_grid(groups, 512), 512, 0, s>>>(q8, qf, w8, wf, to, rows, inputs, outputs, p.m_tiles, p.n_tiles, p.splits); break;
  }
}

template <typename T>
int product(const void *q, const void *qs, const void *w, const void *ws, const void *bias, void *y, long rows, int inputs, int outputs,
            void *workspace, size_t workspace_bytes, hipStream_t s) {
  Plan p = plan_of(rows, inputs, outputs);
  if (p.splits > 1 && (!workspace || workspace_bytes < sizeof(float) * p.splits * static_cast<size_t>(rows) * outputs)) p.splits = 1;
  float *const part = p.splits > 1 ? static_cast<float *>(workspace) : nullptr;
  const Results<T> to{static_cast<T *>(y), static_cast<const T *>(bias), part, rows, outputs};
  launch(p, q, qs, w, ws, to, static_cast<int>(rows), inputs, outputs, s);
  if (part) {
    const long count = rows * outputs;
    if (p.splits > 8) join_parts<T, 8><<<linear_grid((count + 31) / 32, 256), 256, 0, s>>>(part, to.bias, to.y, count, outputs, p.splits);
    else join_parts<T, 1><<<linear_grid((count + 255) / 256, 256), 256, 0, s>>>(part, to.bias, to.y, count, outputs, p.splits);
  }
  return check_launch("block_linear");
}

}  // namespace
}  // namespace mv

using namespace mv;

extern "C" {

size_t mv_block_linear_workspace_bytes(int64_t rows, int inputs, int outputs) {
  if (rows <= 0 || inputs <= 0 || outputs <= 0 || inputs % kBlock) return 0;
  const Plan p = plan_of(rows, inputs, outputs);
  return p.splits > 1 ? sizeof(float) * p.splits * static_cast<size_t>(rows) * outputs : 0;
}

int mv_block_linear(const void *q, const void *q_scales, const void *weight, const void *weight_scales, const void *bias,
                    void *y, int64_t rows, int inputs, int outputs, int dtype, void *workspace, size_t workspace_bytes,
                    void *stream) {
  MV_REQUIRE(dtype == MV_F16 || dtype == MV_BF16, "dtype %d of the output is not float16 or bfloat16", dtype);
  MV_REQUIRE(rows >= 0 && rows < (1L << 31) - 256 && inputs > 0 && outputs >= 0 && outputs < (1L << 31) - 256 && inputs % kBlock == 0,
             "wrong sizes: %ld rows, %d inputs (whole blocks of 128), %d outputs", static_cast<long>(rows), inputs, outputs);
  if (rows == 0 || outputs == 0) return MV_OK;
  MV_REQUIRE(q && q_scales && weight && weight_scales && y, "a tensor is missing");
  MV_REQUIRE(reinterpret_cast<uintptr_t>(q) % 16 == 0 && reinterpret_cast<uintptr_t>(weight) % 16 == 0, "q and weight have to be 16-byte aligned");
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return dtype == MV_F16 ? product<__half>(q, q_scales, weight, weight_scales, bias, y, rows, inputs, outputs, workspace, workspace_bytes, s)
                         : product<__hip_bfloat16>(q, q_scales, weight, weight_scales, bias, y, rows, inputs, outputs, workspace, workspace_bytes, s);
}

}  // extern "C"

// Eight consecutive values of a row: the unit in which the norm, the quantiser and the attention kernels read and write.
#pragma once
#include "common.hpp"

namespace mv {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

// Vectors at the alignment of one element: the compiler emits the same 16-byte instruction as for an aligned address, and
// global memory takes it at any address (rows of odd length, views that start in the middle of a row).
template <typename V, int A> struct __attribute__((packed, aligned(A))) Loose { V v; };

template <typename T> struct Bits;   // element <-> float on raw bits
template <> struct Bits<__half> {
  static __device__ __forceinline__ float up(unsigned short b) { return __half2float(__ushort_as_half(b)); }
};
template <> struct Bits<__hip_bfloat16> {
  static __device__ __forceinline__ float up(unsigned short b) { return __uint_as_float(static_cast<unsigned>(b) << 16); }
};

// out[0..7] = p[0..7], zeros from `left` on
template <typename T> __device__ __forceinline__ void load_tail(const T *p, int left, float (&out)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) out[i] = 0.f;
  if (left <= 0) return;
  float v[7];   // (eight addresses that all exist: one wait instead of a branch for each)
#pragma unroll
  for (int i = 0; i < 7; ++i) v[i] = load(p + min(i, left - 1));
#pragma unroll
  for (int i = 0; i < 7; ++i) out[i] = i < left ? v[i] : 0.f;
}
template <typename T> __device__ __forceinline__ void load8(const T *p, int left, float (&out)[8]) {
  if (left >= 8) {
    const u32x4 r = reinterpret_cast<const Loose<u32x4, 2> *>(p)->v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      out[2 * i] = Bits<T>::up(static_cast<unsigned short>(r[i] & 0xffffu));
      out[2 * i + 1] = Bits<T>::up(static_cast<unsigned short>(r[i] >> 16));
    }
    return;
  }
  load_tail(p, left, out);
}
template <> __device__ __forceinline__ void load8<float>(const float *p, int left, float (&out)[8]) {
  if (left >= 8) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const f32x4 r = reinterpret_cast<const Loose<f32x4, 4> *>(p + 4 * h)->v;
#pragma unroll
      for (int i = 0; i < 4; ++i) out[4 * h + i] = r[i];
    }
    return;
  }
  load_tail(p, left, out);
}

// Two neighbouring values of 16 bits
template <typename T> __device__ __forceinline__ unsigned pack2(float a, float b);
template <> __device__ __forceinline__ unsigned pack2<__half>(float a, float b) {
  typedef _Float16 h2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(unsigned, h2{static_cast<_Float16>(a), static_cast<_Float16>(b)});
}
template <> __device__ __forceinline__ unsigned pack2<__hip_bfloat16>(float a, float b) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  typedef __bf16 b2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(unsigned, __builtin_convertvector(f2{a, b}, b2));
}

template <typename T> __device__ __forceinline__ void store8(T *p, int left, const float (&v)[8]) {
  if (left >= 8) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
    reinterpret_cast<Loose<u32x4, 2> *>(p)->v = r;
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < left) p[i] = store_cast<T>(v[i]);
}
template <> __device__ __forceinline__ void store8<float>(float *p, int left, const float (&v)[8]) {
  if (left >= 8) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const f32x4 r = {v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]};
      reinterpret_cast<Loose<f32x4, 4> *>(p + 4 * h)->v = r;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < left) p[i] = v[i];
}

// Eight elements as they are in memory
template <typename T> struct Raw {
  u32x4 bits[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T *p) {
#pragma unroll
    for (unsigned i = 0; i < sizeof(T) / 2; ++i) bits[i] = reinterpret_cast<const Loose<u32x4, sizeof(T)> *>(p)[i].v;
  }
  __device__ __forceinline__ void values(float (&v)[8]) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(bits[i / 4][i % 4]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = Bits<T>::up(static_cast<unsigned short>(bits[0][i / 2] >> (i % 2 * 16)));
    }
  }
  __device__ __forceinline__ void set(const float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 8; ++i) bits[i / 4][i % 4] = __float_as_uint(v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) bits[0][i] = pack2<T>(v[2 * i], v[2 * i + 1]);
    }
  }
};

// ---- 8-bit blocks --------------------------------------------------------------------------------------
constexpr int kBlock = 128;       // columns that share a scale
constexpr float kE4m3Max = 448.f;
constexpr float kLeastScale = 1.17549435e-38f;   // 2^-126: blocks of zeros, and of values below 448 x 2^-126

// The larger of a and |b|; NaN if either is (a block that holds a NaN stands for NaN throughout).
__device__ __forceinline__ float max_abs(float a, float b) {
  b = fabsf(b);
  return a != a ? a : (b > a || b != b ? b : a);
}
__device__ __forceinline__ float block_scale(float most) {
  const float s = most / kE4m3Max;
  return s < kLeastScale ? kLeastScale : s;   // (NaN stays)
}
// Eight values to e4m3, to nearest even.  |v| <= 448 up to the last bit, which rounds to 448; NaN stays NaN.
__device__ __forceinline__ u32x2 to_e4m3(const float (&v)[8]) {
  u32x2 r;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h], v[4 * h + 1], 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h + 2], v[4 * h + 3], w, true);
    r[h] = static_cast<unsigned>(w);
  }
  return r;
}

// The storage types of the operators on rows
#define MV_FLOATS(dtype, ...)                                                                                    \
  switch (dtype) {                                                                                               \
    case MV_F32: { using T = float; __VA_ARGS__; break; }                                                        \
    case MV_F16: { using T = __half; __VA_ARGS__; break; }                                                       \
    case MV_BF16: { using T = __hip_bfloat16; __VA_ARGS__; break; }                                              \
    default: return ::mv::fail(MV_INVALID_ARGUMENT, "dtype %d is not float32, float16 or bfloat16", (int)(dtype)); \
  }

}  // namespace mv

// Activations of the group norm, and their derivatives, in 32 bits.
#pragma once
#include "common.hpp"

namespace mv {

// (of two branches the derivative at the border is that of the lower one)
template <int Kind> struct Activation {   // MV_NO_ACTIVATION
  static __device__ __forceinline__ float value(float z, float) { return z; }
  static __device__ __forceinline__ float slope(float, float) { return 1.f; }
};
template <> struct Activation<MV_RELU> {
  static __device__ __forceinline__ float value(float z, float) { return z <= 0.f ? 0.f : z; }   // (NaN stays)
  static __device__ __forceinline__ float slope(float z, float) { return z > 0.f ? 1.f : 0.f; }
};
template <> struct Activation<MV_LEAKY_RELU> {
  static __device__ __forceinline__ float value(float z, float low) { return z > 0.f ? z : z * low; }
  static __device__ __forceinline__ float slope(float z, float low) { return z > 0.f ? 1.f : low; }
};
// z p, p = 1 / (1 + 2^(-z log2 e)): exponential and reciprocal of the hardware, 1 ulp each
template <> struct Activation<MV_SILU> {
  static __device__ __forceinline__ float part(float z) {
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504f * z));
  }
  static __device__ __forceinline__ float value(float z, float) { return z * part(z); }
  static __device__ __forceinline__ float slope(float z, float) {
    const float p = part(z);
    return p * fmaf(z, 1.f - p, 1.f);
  }
};
// z P(z), P the normal distribution's: P(-a) = 2^(-a^2 log2(e) / 2) g(a) for a >= 0, g(a) = erfcx(a / sqrt 2) / 2, which
// has no cancellation; z P(z) = max(z, 0) - |z| P(-|z|).  g is a polynomial of degree 9 in t = 1 / (a + 3), without constant
// term, fitted to the least relative error over 0 <= a <= 14 (5e-8; in 32 bits 4e-7); beyond that the exponential is zero.
template <> struct Activation<MV_GELU> {
  static __device__ __forceinline__ float tail(float z, float &bell) {   // P(-|z|); bell = 2^(-z^2 log2(e) / 2)
    const float t = __builtin_amdgcn_rcpf(fabsf(z) + 3.f);
    float g = -4.480641555e+02f;
    g = fmaf(g, t, 8.502715956e+02f);
    g = fmaf(g, t, -5.932856301e+02f);
    g = fmaf(g, t, 1.596182322e+02f);
    g = fmaf(g, t, -1.296933761e+01f);
    g = fmaf(g, t, 9.713217449e+00f);
    g = fmaf(g, t, 3.035284769e+00f);
    g = fmaf(g, t, 1.202176155e+00f);
    g = fmaf(g, t, 3.988646379e-01f);
    bell = __builtin_amdgcn_exp2f(-0.721347520f * z * z);
    return bell * t * g;
  }
  static __device__ __forceinline__ float value(float z, float) {
    float bell;
    const float p = tail(z, bell);
    return fmaf(-fabsf(z), p, z > 0.f ? z : 0.f);   // (NaN: the product's)
  }
  static __device__ __forceinline__ float slope(float z, float) {
    float bell;
    const float p = tail(z, bell);
    return fmaf(z * 0.398942280f, bell, z > 0.f ? 1.f - p : p);
  }
};

// Calls f with the kind of an activation as a constant
template <typename F> void for_activation(int kind, const F &f) {
  using std::integral_constant;
  switch (kind) {
    case MV_RELU: f(integral_constant<int, MV_RELU>()); break;
    case MV_LEAKY_RELU: f(integral_constant<int, MV_LEAKY_RELU>()); break;
    case MV_SILU: f(integral_constant<int, MV_SILU>()); break;
    case MV_GELU: f(integral_constant<int, MV_GELU>()); break;
    default: f(integral_constant<int, MV_NO_ACTIVATION>()); break;
  }
}

}  // namespace mv

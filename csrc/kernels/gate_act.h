// Activations of a gated block (GateAct) and their slopes, in 32 bits.
#pragma once

#include "feedforward.h"
#include "mfma.h"

namespace mcc {
namespace gpu {

constexpr float kLog2e = 1.4426950408889634f;

// The normal distribution function and exp(-v^2 / 2), by the rational form of
// Abramowitz and Stegun 7.1.26: erfc(x) = (a1 t + .. + a5 t^5) exp(-x^2),
// t = 1 / (1 + p x), off by at most 1.5e-7 for x >= 0; halved here.  That bound is
// absolute.  For v < 0 no difference from 1 is formed, so the tail keeps its size, but
// not all digits of bf16: relative to itself the polynomial is off by 5e-5 at
// v = -3, 0.15 % at -5 and 0.65 % at -7, where gelu is -9e-12.  A library erff took 8
// us of 23 at 777 x 1024 x 2736.
__device__ __forceinline__ void normal(float v, float& cdf, float& bell) {
  bell = __builtin_amdgcn_exp2f(-0.5f * kLog2e * v * v);
  const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f * 0.70710678118654752f, fabsf(v), 1.f));
  const float half =
      t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 0.5f * 1.061405429f, 0.5f * -1.453152027f), 0.5f * 1.421413741f),
                       0.5f * -0.284496736f), 0.5f * 0.254829592f) * bell;
  cdf = v < 0.f ? half : 1.f - half;
}

// tanh by Lambert's continued fraction v / (1 + s / (3 + s / (5 + s / (7 + s / 9)))),
// s = v^2, where 1 - 2 r, r = 1 / (exp(2 |v|) + 1), would lose digits; off by up to 5
// units of 2^-24.  With the library's tanhf 1481 x 64 x 9233 took 63.5 us (relu: 37), so 50.
// slope: 1 - tanh^2, which is 4 r (1 - r): the difference from 1 of a tanh that is
// rounded next to 1 would be off by a few percent at |v| = 7 and 0 beyond 9.
template <bool SLOPE = false> __device__ __forceinline__ float tanh_(float v, float* slope = nullptr) {
  const float a = fabsf(v), s = v * v;
  const bool small = a < 0.7f;
  const float r = __builtin_amdgcn_rcpf(small ? fmaf(s, fmaf(s, 15.f, 420.f), 945.f)
                                              : __builtin_amdgcn_exp2f(2.f * kLog2e * a) + 1.f);
  const float f = copysignf(small ? a * fmaf(s, s + 105.f, 945.f) * r : fmaf(-2.f, r, 1.f), v);
  if constexpr (SLOPE) *slope = small ? 1.f - f * f : 4.f * r * (1.f - r);
  return f;
}

template <int A> __device__ __forceinline__ float gate_f(float v) {
  if constexpr (A == GATE_RELU) return v < 0.f ? 0.f : v;  // keeps a NaN
  if constexpr (A == GATE_TANH) return tanh_(v);
  if constexpr (A == GATE_SILU) return v * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-kLog2e * v));
  if constexpr (A == GATE_GELU) {
    float cdf, bell;
    normal(v, cdf, bell);
    return v * cdf;
  }
  return v;
}

// calls f with the activation as a compile-time constant
template <class Fn> __host__ __device__ __forceinline__ void with_gate(int act, Fn&& f) {
  switch (act) {
    case GATE_RELU: f(ActK<GATE_RELU>{}); break;
    case GATE_TANH: f(ActK<GATE_TANH>{}); break;
    case GATE_SILU: f(ActK<GATE_SILU>{}); break;
    case GATE_GELU: f(ActK<GATE_GELU>{}); break;
    default: f(ActK<GATE_NONE>{}); break;
  }
}

// f(v) and f'(v)
template <int A> __device__ __forceinline__ void gate_slope(float v, float& f, float& d) {
  if constexpr (A == GATE_RELU) {
    f = gate_f<A>(v);
    d = v > 0.f ? 1.f : 0.f;
  } else if constexpr (A == GATE_TANH) {
    f = tanh_<true>(v, &d);
  } else if constexpr (A == GATE_SILU) {
    const float s = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-kLog2e * v));
    f = v * s;
    d = s * (1.f + v * (1.f - s));
  } else if constexpr (A == GATE_GELU) {
    float cdf, bell;
    normal(v, cdf, bell);
    f = v * cdf;
    d = fmaf(v, 0.39894228040143268f * bell, cdf);
  } else {
    f = v;
    d = 1.f;
  }
}

}  // namespace gpu
}  // namespace mcc

// Activations of a gated block (GateAct) and their slopes, in 32 bits.
#pragma once

#include "feedforward.h"
#include "mfma.h"

namespace mcc {
namespace gpu {

constexpr float kLog2e = 1.4426950408889634f;

template <int A> __device__ __forceinline__ float gate_f(float v) {
  if constexpr (A == GATE_RELU) return v < 0.f ? 0.f : v;  // keeps a NaN
  if constexpr (A == GATE_TANH) return tanhf(v);
  if constexpr (A == GATE_SILU) return v / (1.f + __builtin_amdgcn_exp2f(-kLog2e * v));
  if constexpr (A == GATE_GELU) return 0.5f * v * (1.f + erff(v * 0.70710678118654752f));
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
    f = tanhf(v);
    d = 1.f - f * f;
  } else if constexpr (A == GATE_SILU) {
    const float s = 1.f / (1.f + __builtin_amdgcn_exp2f(-kLog2e * v));
    f = v * s;
    d = s * (1.f + v * (1.f - s));
  } else if constexpr (A == GATE_GELU) {
    const float c = 0.5f * (1.f + erff(v * 0.70710678118654752f));
    f = v * c;
    d = c + v * (0.39894228040143268f * __builtin_amdgcn_exp2f(-0.5f * kLog2e * v * v));
  } else {
    f = v;
    d = 1.f;
  }
}

}  // namespace gpu
}  // namespace mcc

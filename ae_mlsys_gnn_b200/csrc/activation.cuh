// Activations of the linear layers' epilogue, in fp32.
#pragma once
#include <cuda_runtime.h>
#include <type_traits>
#include "../../include/gnn_b200.h"

namespace gnn {

// 1 - Phi(|z|) of the normal distribution for the gelu of 16-bit results, and exp(-z^2 / 2), which
// its derivative needs: Abramowitz & Stegun, Handbook of Mathematical Functions, 7.1.26,
//   erfc(x) ~ (a1 t + ... + a5 t^5) exp(-x^2), t = 1 / (1 + 0.3275911 x), off by at most 1.5e-7
// (a 16-bit result's half step is 2^-12 of the value at best), at half the instructions of erff.
__device__ __forceinline__ float normal_tail(float z, float& gauss) {
  const float x = fabsf(z) * 0.70710678118654752f;
  const float t = __fdividef(1.f, fmaf(0.3275911f, x, 1.f));
  gauss = __expf(-x * x);
  float p = fmaf(1.061405429f, t, -1.453152027f);
  p = fmaf(p, t, 1.421413741f);
  p = fmaf(p, t, -0.284496736f);
  p = fmaf(p, t, 0.254829592f);
  return 0.5f * p * t * gauss;
}

// y = act(z) for one activation; FINE: the result is kept in fp32
template <int ACT, bool FINE>
__device__ __forceinline__ float act_one(float z, float slope) {
  if constexpr (ACT == GNN_ACT_RELU) return z < 0.f ? 0.f : z;  // a NaN stays one
  else if constexpr (ACT == GNN_ACT_LEAKY_RELU) return z > 0.f ? z : z * slope;
  else if constexpr (ACT == GNN_ACT_ELU) return z > 0.f ? z : expm1f(z);
  else if constexpr (ACT == GNN_ACT_GELU && FINE) return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
  else if constexpr (ACT == GNN_ACT_GELU) {
    float gauss;
    const float tail = normal_tail(z, gauss);
    return z * (z > 0.f ? 1.f - tail : tail);
  } else if constexpr (ACT == GNN_ACT_SILU) return __fdividef(z, 1.f + __expf(-z));
  else return z;
}

// act'(z); at the corner of relu and leaky_relu the slope of the negative side.  gelu and silu have
// reached their limits long before |z| = 100; beyond it (a z that overflowed its 16-bit type, say) the
// products of z with a zero are kept finite.
template <int ACT, bool FINE>
__device__ __forceinline__ float slope_one(float z, float slope) {
  const float near = fminf(fmaxf(z, -100.f), 100.f);
  if constexpr (ACT == GNN_ACT_RELU) return z > 0.f ? 1.f : 0.f;
  else if constexpr (ACT == GNN_ACT_LEAKY_RELU) return z > 0.f ? 1.f : slope;
  else if constexpr (ACT == GNN_ACT_ELU) return z > 0.f ? 1.f : __expf(z);
  else if constexpr (ACT == GNN_ACT_GELU && FINE)
    return 0.5f * (1.f + erff(z * 0.70710678118654752f)) + near * 0.39894228040143268f * __expf(-0.5f * z * z);
  else if constexpr (ACT == GNN_ACT_GELU) {
    float gauss;
    const float tail = normal_tail(z, gauss);
    return fmaf(near * 0.39894228040143268f, gauss, z > 0.f ? 1.f - tail : tail);
  } else if constexpr (ACT == GNN_ACT_SILU) {
    const float s = __fdividef(1.f, 1.f + __expf(-z));  // 0 where __expf overflows to infinity
    return s * (1.f + near * (1.f - s));
  } else return 1.f;
}

// Calls f(std::integral_constant) for an activation: one branch for all values that f handles, so that
// only one activation's instructions are fetched.
template <class F>
__device__ __forceinline__ void with_act(int act, F&& f) {
  switch (act) {
    case GNN_ACT_RELU: f(std::integral_constant<int, GNN_ACT_RELU>{}); break;
    case GNN_ACT_LEAKY_RELU: f(std::integral_constant<int, GNN_ACT_LEAKY_RELU>{}); break;
    case GNN_ACT_ELU: f(std::integral_constant<int, GNN_ACT_ELU>{}); break;
    case GNN_ACT_GELU: f(std::integral_constant<int, GNN_ACT_GELU>{}); break;
    case GNN_ACT_SILU: f(std::integral_constant<int, GNN_ACT_SILU>{}); break;
    default: break;
  }
}

// v[i] = act(v[i])
template <bool FINE, int N>
__device__ __forceinline__ void apply_act(float (&v)[N], int act, float slope) {
  with_act(act, [&](auto a) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = act_one<decltype(a)::value, FINE>(v[i], slope);
  });
}
// v[i] *= act'(z[i])
template <bool FINE, int N>
__device__ __forceinline__ void apply_act_slope(float (&v)[N], const float (&z)[N], int act, float slope) {
  with_act(act, [&](auto a) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] *= slope_one<decltype(a)::value, FINE>(z[i], slope);
  });
}
template <bool FINE>
__device__ __forceinline__ float act_value(float z, int act, float slope) {
  float v[1] = {z};
  apply_act<FINE>(v, act, slope);
  return v[0];
}

}  // namespace gnn

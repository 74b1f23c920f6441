// The activation functions of a linear layer's epilogue and their derivatives, in FP32.
#pragma once
#include <cuda_runtime.h>
#include <type_traits>

namespace i8m {

enum Activation : int { ACT_NONE = 0, ACT_RELU = 1, ACT_RELU2 = 2, ACT_GELU = 3, ACT_GELU_TANH = 4, ACT_SILU = 5 };
constexpr int ACTIVATIONS = 6;

// 2^v and 1 / v on the special-function unit, good to a few units in the last place; 1 / inf is 0.
__device__ __forceinline__ float exp2_fast(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float reciprocal_fast(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
constexpr float LOG2_E = 1.4426950408889634f;
__device__ __forceinline__ float logistic(float v) { return reciprocal_fast(1.f + exp2_fast(-LOG2_E * v)); }

// Normal distribution function and density.  For a = |z| and t = 1 / (1 + 0.3 a), the lower tail Phi(-a) is
// exp(-a^2 / 2) t P(t): Phi(-a) exp(a^2 / 2) falls like 1 / a, so it is t times a smooth function, here a polynomial of degree 7
// fitted for the least relative error over 0 <= a <= 14, where the tail leaves FP32's range: 1.5e-7 in exact arithmetic, 5e-7
// with FP32 roundings over a grid of 200 000 points.  The exponential is the density's as well.
struct NormalAt { float cdf, pdf; };
__device__ __forceinline__ NormalAt normal_at(float z) {
  const float e = exp2_fast(-0.5f * LOG2_E * z * z);
  const float t = reciprocal_fast(fmaf(0.3f, fabsf(z), 1.f));
  float p = 0.0356747769f;
  p = fmaf(p, t, -0.157203108f);
  p = fmaf(p, t, 0.20635353f);
  p = fmaf(p, t, -0.0536836721f);
  p = fmaf(p, t, 0.128561646f);
  p = fmaf(p, t, 0.0999134853f);
  p = fmaf(p, t, 0.120753959f);
  p = fmaf(p, t, 0.119629301f);
  const float tail = e * t * p;
  return {z < 0.f ? tail : 1.f - tail, 0.39894228040143268f * e};
}

constexpr float GELU_TANH_C = 2.f * 0.79788456080286536f;     // 2 sqrt(2 / pi)
constexpr float GELU_TANH_K = GELU_TANH_C * 0.044715f;

template <int ACT>
__device__ __forceinline__ float activate(float z) {
  if constexpr (ACT == ACT_RELU) return z < 0.f ? 0.f : z;              // NaN stays NaN
  if constexpr (ACT == ACT_RELU2) return z < 0.f ? 0.f : z * z;
  if constexpr (ACT == ACT_GELU) return z * normal_at(z).cdf;
  // 1/2 (1 + tanh u) is the logistic function of 2 u
  if constexpr (ACT == ACT_GELU_TANH) return z * logistic(z * fmaf(GELU_TANH_K, z * z, GELU_TANH_C));
  if constexpr (ACT == ACT_SILU) return z * logistic(z);
  return z;
}
template <int ACT>
__device__ __forceinline__ float derivative(float z) {
  if constexpr (ACT == ACT_RELU) return z > 0.f ? 1.f : (z <= 0.f ? 0.f : z);
  if constexpr (ACT == ACT_RELU2) return z < 0.f ? 0.f : 2.f * z;
  if constexpr (ACT == ACT_GELU) {
    const NormalAt n = normal_at(z);
    return fmaf(z, n.pdf, n.cdf);
  }
  if constexpr (ACT == ACT_GELU_TANH) {
    const float s = logistic(z * fmaf(GELU_TANH_K, z * z, GELU_TANH_C));
    const float slope = fmaf(3.f * GELU_TANH_K, z * z, GELU_TANH_C);
    return fmaf(z * s * (1.f - s), slope, s);
  }
  if constexpr (ACT == ACT_SILU) {
    const float s = logistic(z);
    return fmaf(z * s, 1.f - s, s);
  }
  return 1.f;
}
// Calls f(std::integral_constant<int, ACT>) for the run-time code `act`.
template <class F>
__device__ __forceinline__ void with_activation(int act, F&& f) {
  switch (act) {
    case ACT_RELU: f(std::integral_constant<int, ACT_RELU>{}); break;
    case ACT_RELU2: f(std::integral_constant<int, ACT_RELU2>{}); break;
    case ACT_GELU: f(std::integral_constant<int, ACT_GELU>{}); break;
    case ACT_GELU_TANH: f(std::integral_constant<int, ACT_GELU_TANH>{}); break;
    case ACT_SILU: f(std::integral_constant<int, ACT_SILU>{}); break;
    default: f(std::integral_constant<int, ACT_NONE>{}); break;
  }
}

}  // namespace i8m

// The activation functions of a linear layer's epilogue and their derivatives, in FP32.
#pragma once
#include <cuda_runtime.h>

namespace i8m {

enum Activation : int { ACT_NONE = 0, ACT_RELU = 1, ACT_RELU2 = 2, ACT_GELU = 3, ACT_GELU_TANH = 4, ACT_SILU = 5 };
constexpr int ACTIVATIONS = 6;

__device__ __forceinline__ float logistic(float v) { return 1.f / (1.f + expf(-v)); }

// Normal distribution function through the complementary error function, which keeps its relative precision in the
// lower tail.
__device__ __forceinline__ float normal_cdf(float z) { return 0.5f * erfcf(-0.70710678118654752f * z); }

constexpr float GELU_TANH_C = 0.79788456080286536f;     // sqrt(2 / pi)
constexpr float GELU_TANH_K = 0.044715f;

template <int ACT>
__device__ __forceinline__ float activate(float z) {
  if constexpr (ACT == ACT_RELU) return z < 0.f ? 0.f : z;              // NaN stays NaN
  if constexpr (ACT == ACT_RELU2) return z < 0.f ? 0.f : z * z;
  if constexpr (ACT == ACT_GELU) return z * normal_cdf(z);
  // 1/2 (1 + tanh u) is the logistic function of 2 u
  if constexpr (ACT == ACT_GELU_TANH) return z * logistic(2.f * GELU_TANH_C * fmaf(GELU_TANH_K * z * z, z, z));
  if constexpr (ACT == ACT_SILU) return z * logistic(z);
  return z;
}
template <int ACT>
__device__ __forceinline__ float derivative(float z) {
  if constexpr (ACT == ACT_RELU) return z > 0.f ? 1.f : (z <= 0.f ? 0.f : z);
  if constexpr (ACT == ACT_RELU2) return z < 0.f ? 0.f : 2.f * z;
  if constexpr (ACT == ACT_GELU) return fmaf(z, 0.39894228040143268f * expf(-0.5f * z * z), normal_cdf(z));
  if constexpr (ACT == ACT_GELU_TANH) {
    const float s = logistic(2.f * GELU_TANH_C * fmaf(GELU_TANH_K * z * z, z, z));
    const float slope = 2.f * GELU_TANH_C * fmaf(3.f * GELU_TANH_K * z, z, 1.f);
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

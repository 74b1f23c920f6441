// The activation functions of a linear layer's epilogue, on pairs, and their derivatives, in FP32.
#pragma once
#include "vectors.cuh"
#include <type_traits>

namespace i8m {

enum Activation : int { ACT_NONE = 0, ACT_RELU = 1, ACT_RELU2 = 2, ACT_GELU = 3, ACT_GELU_TANH = 4, ACT_SILU = 5 };
constexpr int ACTIVATIONS = 6;

// 2^v and 1 / v on the special-function unit, good to a few units in the last place; 1 / inf is 0, and results below 2^-126
// are 0: silu below z = -87.3, where its value is -1e-36, and gelu_tanh below -10.0, where it is -1.2e-37.
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

__device__ __forceinline__ float max_nan(float a, float b) {      // a NaN stays one
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Normal distribution: the lower tail Phi(-a) and exp(-a^2 / 2) for two a = min(|z|, 30) (beyond 14 the tail is zero in FP32).
// With t = 1 / (1 + 0.3 a), Phi(-a) is exp(-a^2 / 2) t P(t): Phi(-a) exp(a^2 / 2) falls like 1 / a, so it is t times a smooth
// function, here a polynomial of degree 7 fitted for the least relative error over 0 <= a <= 14: t P(t) is good to 1.5e-7 in
// exact arithmetic and 5e-7 with FP32 roundings, over a grid of 400 000 points.  The exponential adds the roundings of its
// argument, which grow with a^2 / 2: the tail's relative error is 6e-7 up to a = 3, 2e-6 up to 6, 3.3e-6 up to 9 and 8e-6 up to
// 12.9, where the tail is 2e-38.  Ten issue slots per element with the pairs, twenty without.
struct NormalTail { unsigned long long tail, density; };
__device__ __forceinline__ NormalTail normal_tail(unsigned long long a) {
  const unsigned long long s = mul2(mul2(a, both(-0.5f * LOG2_E)), a), q = fma2(both(0.3f), a, both(1.f));
  const unsigned long long e = pair(exp2_fast(lane0(s)), exp2_fast(lane1(s)));
  const unsigned long long t = pair(reciprocal_fast(lane0(q)), reciprocal_fast(lane1(q)));
  unsigned long long p = both(0.0356747769f);
  p = fma2(p, t, both(-0.157203108f));
  p = fma2(p, t, both(0.20635353f));
  p = fma2(p, t, both(-0.0536836721f));
  p = fma2(p, t, both(0.128561646f));
  p = fma2(p, t, both(0.0999134853f));
  p = fma2(p, t, both(0.120753959f));
  p = fma2(p, t, both(0.119629301f));
  return {mul2(mul2(e, t), p), e};
}
__device__ __forceinline__ float bounded_magnitude(float z) { return fminf(fabsf(z), 30.f); }

constexpr float GELU_TANH_C = 2.f * 0.79788456080286536f;     // 2 sqrt(2 / pi)
constexpr float GELU_TANH_K = GELU_TANH_C * 0.044715f;

// 1 / (1 + 2^v) of a pair: the logistic function of -v log 2
__device__ __forceinline__ unsigned long long gate2(unsigned long long v) {
  const unsigned long long d = add2(pair(exp2_fast(lane0(v)), exp2_fast(lane1(v))), both(1.f));
  return pair(reciprocal_fast(lane0(d)), reciprocal_fast(lane1(d)));
}
template <int ACT>
__device__ __forceinline__ unsigned long long activate(unsigned long long z) {
  const float z0 = lane0(z), z1 = lane1(z);
  if constexpr (ACT == ACT_RELU) return pair(max_nan(z0, 0.f), max_nan(z1, 0.f));
  if constexpr (ACT == ACT_RELU2) {
    const unsigned long long p = pair(max_nan(z0, 0.f), max_nan(z1, 0.f));
    return mul2(p, p);
  }
  if constexpr (ACT == ACT_GELU) {
    // z Phi(z) = max(z, 0) - |z| Phi(-|z|)
    const unsigned long long a = pair(bounded_magnitude(z0), bounded_magnitude(z1));
    return fma2(mul2(a, both(-1.f)), normal_tail(a).tail, pair(max_nan(z0, 0.f), max_nan(z1, 0.f)));
  }
  // 1/2 (1 + tanh u) is the logistic function of 2 u
  if constexpr (ACT == ACT_GELU_TANH)
    return mul2(z, gate2(mul2(z, fma2(both(-LOG2_E * GELU_TANH_K), mul2(z, z), both(-LOG2_E * GELU_TANH_C)))));
  if constexpr (ACT == ACT_SILU) return mul2(z, gate2(mul2(z, both(-LOG2_E))));
  return z;
}
// z as a factor of s (1 - s), s the logistic function of z or of a cubic in it: bounded, and its square as well, so that the
// product is zero where s is 0 or 1 to the last bit (from |z| = 90 on), at infinities too - a kept pre-activation is one where the
// forward pass's FP32 value is beyond the kept type.  A NaN is lost here and stays in s.
// One instruction, the smaller magnitude under the product of both signs: silu's slopes for the bias gradient of 8192 x 14336
// take 89.6 us, 91.6 with a minimum and a maximum, 88.5 without a bound; gelu_tanh's 99.4, 101.4, 98.6.
__device__ __forceinline__ float bounded_value(float z) {
  float r;
  asm("min.xorsign.abs.f32 %0, %1, %2;" : "=f"(r) : "f"(z), "f"(1e15f));
  return r;
}
template <int ACT>
__device__ __forceinline__ unsigned long long derivative(unsigned long long z) {
  const float z0 = lane0(z), z1 = lane1(z);
  if constexpr (ACT == ACT_RELU) return pair(z0 > 0.f ? 1.f : (z0 <= 0.f ? 0.f : z0), z1 > 0.f ? 1.f : (z1 <= 0.f ? 0.f : z1));
  if constexpr (ACT == ACT_RELU2) return mul2(pair(max_nan(z0, 0.f), max_nan(z1, 0.f)), both(2.f));
  if constexpr (ACT == ACT_GELU) {
    const NormalTail n = normal_tail(pair(bounded_magnitude(z0), bounded_magnitude(z1)));
    const float t0 = lane0(n.tail), t1 = lane1(n.tail);
    // the bounded z: where it differs the density is zero (and a NaN stays one)
    const unsigned long long b = pair(max_nan(-30.f, z0 > 30.f ? 30.f : z0), max_nan(-30.f, z1 > 30.f ? 30.f : z1));
    return fma2(mul2(b, both(0.39894228040143268f)), n.density, pair(z0 < 0.f ? t0 : 1.f - t0, z1 < 0.f ? t1 : 1.f - t1));
  }
  if constexpr (ACT == ACT_GELU_TANH) {
    const unsigned long long b = pair(bounded_value(z0), bounded_value(z1)), q = mul2(b, b);
    const unsigned long long s = gate2(mul2(z, fma2(both(-LOG2_E * GELU_TANH_K), q, both(-LOG2_E * GELU_TANH_C))));
    const unsigned long long slope = fma2(both(3.f * GELU_TANH_K), q, both(GELU_TANH_C));
    return fma2(mul2(mul2(b, s), fma2(s, both(-1.f), both(1.f))), slope, s);
  }
  if constexpr (ACT == ACT_SILU) {
    const unsigned long long s = gate2(mul2(z, both(-LOG2_E))), b = pair(bounded_value(z0), bounded_value(z1));
    return fma2(mul2(b, s), fma2(s, both(-1.f), both(1.f)), s);
  }
  return both(1.f);
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

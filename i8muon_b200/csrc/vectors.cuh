// Eight consecutive elements of any of the three types as 16-byte vectors, and FP32 arithmetic on pairs.
#pragma once
#include "epi_float.cuh"

namespace i8m {

// packed two-lane FP32 arithmetic (sm_100): one issue slot for two IEEE operations
__device__ __forceinline__ unsigned long long pack2(uint32_t lo, uint32_t hi) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
  return r;
}
__device__ __forceinline__ unsigned long long add2(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b,
                                                   unsigned long long c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ float lane0(unsigned long long v) { return __uint_as_float(uint32_t(v)); }
__device__ __forceinline__ float lane1(unsigned long long v) { return __uint_as_float(uint32_t(v >> 32)); }
__device__ __forceinline__ unsigned long long mul2(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ unsigned long long pair(float lo, float hi) { return pack2(__float_as_uint(lo), __float_as_uint(hi)); }
__device__ __forceinline__ unsigned long long both(float v) { return pair(v, v); }

template <typename In>
__device__ __forceinline__ void unpack8(const uint4 raw, float (&v)[8]) {
  const In* e = reinterpret_cast<const In*>(&raw);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = widen<In>(e[j]);
}
// eight consecutive input elements (16-byte aligned): one vector load for 16-bit types, two for FP32
template <typename In>
__device__ __forceinline__ void load8(const In* p, float (&v)[8]) {
  if constexpr (sizeof(In) == 4) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    unpack8<In>(*reinterpret_cast<const uint4*>(p), v);
  }
}
// Eight consecutive values as one vector, p on its size (32 bytes for FP32: two 16-byte stores leave half-written sectors to L2,
// and restoring 8192 x 4096 FP32 activations took 39.9 us).
template <typename E>
__device__ __forceinline__ void store8(E* p, const float (&v)[8]) {
  if constexpr (sizeof(E) == 4) {
    asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]),
                 "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]) : "memory");
  } else {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack2<E>(v[0], v[1]), pack2<E>(v[2], v[3]), pack2<E>(v[4], v[5]), pack2<E>(v[6], v[7]));
  }
}

}  // namespace i8m

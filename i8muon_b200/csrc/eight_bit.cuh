// Activations kept in eight bits for the backward pass.
//
// A row is cut into groups of 32 consecutive elements (the last one may be short).  A group with the largest magnitude
// top has one exponent e, the smallest integer with top <= M 2^e (M = 127 for INT8, 448 for E4M3; e >= -127), stored as
// the byte e + 127.  A code is x 2^-e rounded to the nearest integer or E4M3 value, ties to even, and stands for code 2^e.
//
// Why a power of two: x 2^-e and code 2^e are exact, so the codes are the same however they are computed, and a kept
// value has at most eight significant bits, which FP16, BF16 and FP32 all hold: restoring rounds nothing.  The price is
// at most one bit of an INT8 code against a scale of top / 127 (half a step is at most top / 127), none of E4M3, whose
// relative step does not depend on the scale.  Why 32: one thread of a product's epilogue holds 32 columns of a row, a
// warp one per lane, and a channel ten times larger than the others costs precision to its 31 neighbours only.
//
// Beside the largest number of a type, rounding up would leave the type: there the code below is taken (63 2^e, 240 2^e).
// The pre-activations that a product's epilogue writes are FP32 values, within no 16-bit type's range: they are kept in FP32's
// range and read by linear_dz_kernel alone.  A finite one beside 2^128 may read back as an infinity; slopes are at their limits there.
// A group that holds an infinity or a NaN has the byte 255 and reads back as NaN throughout: a loss scaler sees it.
// Codes behind the end of a row are zero.
#pragma once
#include "epi_float.cuh"

namespace i8m {

enum EightFormat : int { EIGHT_INT8 = 0, EIGHT_E4M3 = 1 };
constexpr int EIGHT_GROUP = 32;
constexpr uint32_t EIGHT_NAN = 255u;

// Exponent byte of a group from the largest bit pattern of its magnitudes (sign bits cleared): integer order is the
// order of the magnitudes, with infinity and NaN above all numbers.  127 = 0x7E0000 (mantissa) x 2^6, 448 = 0x600000 x 2^8:
// adding what the mantissa lacks to 2^23 carries into the exponent exactly where top exceeds M 2^e.
template <int FORMAT>
__device__ __forceinline__ uint32_t eight_exponent(uint32_t top) {
  if (top >= 0x7f800000u) return EIGHT_NAN;
  const int e = FORMAT == EIGHT_INT8 ? int((top + 0x1ffffu) >> 23) - 6 : int((top + 0x1fffffu) >> 23) - 8;
  return uint32_t(e > 0 ? e : 0);
}
// max(top, |a|, |b|) in one instruction; a NaN anywhere stays one.  Its bits are what eight_exponent takes.
__device__ __forceinline__ float top_of(float top, float a, float b) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(top), "f"(a), "f"(b));
  return r;
}
// 2^-e (a normal number: bytes of finite groups end at 249; zero for the others) and 2^e.
__device__ __forceinline__ float eight_inverse(uint32_t byte) { return __uint_as_float((254u - min(byte, 254u)) << 23); }
__device__ __forceinline__ float eight_step(uint32_t byte) {
  return __uint_as_float(byte == 0u ? 0x00400000u : byte == EIGHT_NAN ? 0x7fc00000u : byte << 23);
}

// The groups of type E in which rounding up may pass the type's largest number are those with the exponent of that number;
// every finite element above LIMIT is in one of them, and LIMIT is a code's value there.
template <typename E, int FORMAT>
struct EightTop {
  static constexpr bool HALF = std::is_same<E, __half>::value;
  static constexpr int EXPONENT = FORMAT == EIGHT_INT8 ? (HALF ? 10 : 122) : (HALF ? 8 : 120);
  static constexpr uint32_t BYTE = uint32_t(EXPONENT + 127);
  static __device__ __forceinline__ float clip(float x) {
    const float limit = (FORMAT == EIGHT_INT8 ? 63.f : 240.f) * __uint_as_float(BYTE << 23);
    return fminf(fmaxf(x, -limit), limit);
  }
};

// Four codes of x[0..3] packed into a word, lowest byte first.
template <int FORMAT>
__device__ __forceinline__ uint32_t eight_encode4(float x0, float x1, float x2, float x3, float inverse) {
  if constexpr (FORMAT == EIGHT_INT8) {
    // adding 1.5 2^23 rounds to an integer, to nearest and ties to even, and leaves it in the low bits
    constexpr float MAGIC = 12582912.f;
    const uint32_t a = __float_as_uint(fmaf(x0, inverse, MAGIC)), b = __float_as_uint(fmaf(x1, inverse, MAGIC));
    const uint32_t c = __float_as_uint(fmaf(x2, inverse, MAGIC)), d = __float_as_uint(fmaf(x3, inverse, MAGIC));
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
  } else {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x0 * inverse, x1 * inverse), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x2 * inverse, x3 * inverse), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
  }
}
// The four values that a word of codes stands for.
template <int FORMAT>
__device__ __forceinline__ void eight_decode4(uint32_t codes, float step, float (&v)[4]) {
  if constexpr (FORMAT == EIGHT_INT8) {
    // code + 128 into the low mantissa bits of 2^23, minus 2^23 + 128: exact, and no conversion instruction
    const uint32_t u = codes ^ 0x80808080u;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (__uint_as_float(__byte_perm(u, 0x4B000000u, 0x7440u + i)) - 8388736.f) * step;
  } else {
    const __half2 lo = __half2(__nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(codes & 0xffffu), __NV_E4M3));
    const __half2 hi = __half2(__nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(codes >> 16), __NV_E4M3));
    const float2 a = __half22float2(lo), b = __half22float2(hi);
    v[0] = a.x * step; v[1] = a.y * step; v[2] = b.x * step; v[3] = b.y * step;
  }
}
template <int FORMAT>
__device__ __forceinline__ uint8_t eight_encode1(float x, float inverse) {
  return uint8_t(eight_encode4<FORMAT>(x, 0.f, 0.f, 0.f, inverse));
}
template <int FORMAT>
__device__ __forceinline__ float eight_decode1(uint8_t code, float step) {
  float v[4];
  eight_decode4<FORMAT>(code, step, v);
  return v[0];
}

}  // namespace i8m

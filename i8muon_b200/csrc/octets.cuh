// Octets (eight consecutive elements) of rows that start anywhere.
//
// A row of a tensor with an odd width starts at any element, so that its octets do not lie on 16 bytes.  Reading one means
// reading the two (FP32: three) aligned 16-byte pieces that hold it and shifting; all octets of a row are shifted alike, so the
// selections are uniform.  Writing means building aligned pieces from an octet and its left neighbour's, one lane away.
// Single elements are loaded at the ends of a tensor and stored at the ends of a warp's run.
#pragma once
#include "vectors.cuh"

namespace i8m {

// Eight elements as they lie in memory.
template <typename E>
struct Octet {
  static constexpr int WORDS = int(sizeof(E)) * 2;
  uint32_t q[WORDS];
  // elements 2 k and 2 k + 1
  __device__ __forceinline__ unsigned long long get(int k) const {
    if constexpr (WORDS == 8) {
      return pack2(q[2 * k], q[2 * k + 1]);
    } else {
      const float2 f = unpack2<E>(q[k]);
      return pair(f.x, f.y);
    }
  }
  __device__ __forceinline__ void load(const E* p) {          // on 16 bytes
#pragma unroll
    for (int k = 0; k < WORDS / 4; ++k) {
      const uint4 w = reinterpret_cast<const uint4*>(p)[k];
      q[4 * k] = w.x; q[4 * k + 1] = w.y; q[4 * k + 2] = w.z; q[4 * k + 3] = w.w;
    }
  }
  __device__ __forceinline__ void pack(const float (&v)[8]) {
    if constexpr (WORDS == 8) {
#pragma unroll
      for (int k = 0; k < 8; ++k) q[k] = __float_as_uint(v[k]);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) q[k] = pack2<E>(v[2 * k], v[2 * k + 1]);
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int k = 0; k < WORDS; ++k) q[k] = 0u;
  }
  __device__ __forceinline__ E element(int j) const {         // j known at compile time
    if constexpr (WORDS == 8) {
      return E(__uint_as_float(q[j]));
    } else {
      const uint16_t h = uint16_t(j & 1 ? q[j >> 1] >> 16 : q[j >> 1]);
      return *reinterpret_cast<const E*>(&h);
    }
  }
  // elements from n on become zero
  __device__ __forceinline__ void cut(int n) {
#pragma unroll
    for (int k = 0; k < WORDS; ++k) {
      if constexpr (WORDS == 8) q[k] = k < n ? q[k] : 0u;
      else q[k] &= (2 * k < n ? 0xffffu : 0u) | (2 * k + 1 < n ? 0xffff0000u : 0u);
    }
  }
};

// w[0 .. N) <- w[shift .. shift + N), 0 <= shift <= 3.
template <int N, int M>
__device__ __forceinline__ void shift_words(uint32_t (&w)[M], uint32_t shift) {
  static_assert(M >= N + 3, "three words behind");
  const bool two = shift & 2u, one = shift & 1u;
#pragma unroll
  for (int i = 0; i < N + 1; ++i) w[i] = two ? w[i + 2] : w[i];
#pragma unroll
  for (int i = 0; i < N; ++i) w[i] = one ? w[i + 1] : w[i];
}

// n of the eight elements at p exist (none if n <= 0), the others read as zero; the tensor reaches from `begin` to `end`, and
// nothing outside is read.
template <typename E>
__device__ __forceinline__ void load_any(Octet<E>& o, const E* p, int n, const E* begin, const E* end) {
  constexpr int WORDS = Octet<E>::WORDS, PIECES = WORDS / 4 + 1;
  o.clear();
  if (n <= 0) return;
  const uintptr_t at = reinterpret_cast<uintptr_t>(p);
  const uint32_t off = uint32_t(at & 15u);
  const uintptr_t base = at - off;
  const int pieces = off == 0 ? PIECES - 1 : PIECES;
  if (base >= reinterpret_cast<uintptr_t>(begin) && base + 16u * pieces <= reinterpret_cast<uintptr_t>(end)) {
    uint32_t w[4 * PIECES + 3];
#pragma unroll
    for (int k = 0; k < PIECES; ++k) {
      if (k < pieces) {
        const uint4 v = reinterpret_cast<const uint4*>(base)[k];
        w[4 * k] = v.x; w[4 * k + 1] = v.y; w[4 * k + 2] = v.z; w[4 * k + 3] = v.w;
      } else {
        w[4 * k] = w[4 * k + 1] = w[4 * k + 2] = w[4 * k + 3] = 0u;
      }
    }
    w[4 * PIECES] = w[4 * PIECES + 1] = w[4 * PIECES + 2] = 0u;
    if constexpr (WORDS == 8) {
      shift_words<8>(w, off >> 2);
#pragma unroll
      for (int k = 0; k < 8; ++k) o.q[k] = w[k];
    } else {
      shift_words<5>(w, off >> 2);
#pragma unroll
      for (int k = 0; k < 4; ++k) o.q[k] = __funnelshift_r(w[k], w[k + 1], (off & 2u) * 8u);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (j >= n) continue;
      if constexpr (WORDS == 8) o.q[j] = __float_as_uint(p[j]);
      else o.q[j >> 1] |= uint32_t(*reinterpret_cast<const uint16_t*>(p + j)) << (16 * (j & 1));
    }
  }
  if (n < 8) o.cut(n);
}

// Eight elements at p without a branch, for loads that shall be on their way together: all pieces that load_inside_fits names exist.
template <typename E>
__device__ __forceinline__ bool load_inside_fits(const E* first, const E* last, const E* begin, const E* end) {
  constexpr uintptr_t BYTES = 16 * (Octet<E>::WORDS / 4 + 1);
  return (reinterpret_cast<uintptr_t>(first) & ~uintptr_t(15)) >= reinterpret_cast<uintptr_t>(begin) &&
         (reinterpret_cast<uintptr_t>(last) & ~uintptr_t(15)) + BYTES <= reinterpret_cast<uintptr_t>(end);
}
template <typename E>
__device__ __forceinline__ void load_inside(uint32_t (&w)[Octet<E>::WORDS + 7], const E* p) {
  const uint4* base = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(p) & ~uintptr_t(15));
#pragma unroll
  for (int k = 0; k < Octet<E>::WORDS / 4 + 1; ++k) {
    const uint4 v = base[k];
    w[4 * k] = v.x; w[4 * k + 1] = v.y; w[4 * k + 2] = v.z; w[4 * k + 3] = v.w;
  }
  w[Octet<E>::WORDS + 4] = w[Octet<E>::WORDS + 5] = w[Octet<E>::WORDS + 6] = 0u;
}
template <typename E>
__device__ __forceinline__ void shift_inside(Octet<E>& o, uint32_t (&w)[Octet<E>::WORDS + 7], const E* p, int n) {
  const uint32_t off = uint32_t(reinterpret_cast<uintptr_t>(p) & 15u);
  if constexpr (Octet<E>::WORDS == 8) {
    shift_words<8>(w, off >> 2);
#pragma unroll
    for (int k = 0; k < 8; ++k) o.q[k] = w[k];
  } else {
    shift_words<5>(w, off >> 2);
#pragma unroll
    for (int k = 0; k < 4; ++k) o.q[k] = __funnelshift_r(w[k], w[k + 1], (off & 2u) * 8u);
  }
  if (n < 8) o.cut(n);
}

// Stores the n (0 .. 8) first elements of every lane's octet.  All lanes call it; lane l's octet starts 8 l elements behind lane
// 0's, and only the last lane that has elements may have fewer than eight.
template <typename E>
__device__ __forceinline__ void store_any(E* p, int n, const Octet<E>& o) {
  constexpr int WORDS = Octet<E>::WORDS;
  const int lane = threadIdx.x & 31;
  const uint32_t off = uint32_t(reinterpret_cast<uintptr_t>(p) & 15u);      // the same in all lanes
  const int tail = off == 0 ? 8 : 8 - int(off / sizeof(E));                // elements from here on belong to the next lane's
  uint32_t w[WORDS + 4 + 3];
  // words: the last piece of the left neighbour, this lane's, and room for shift_words
#pragma unroll
  for (int k = 0; k < 4; ++k) w[k] = __shfl_up_sync(0xffffffffu, o.q[WORDS - 4 + k], 1);
#pragma unroll
  for (int k = 0; k < WORDS; ++k) w[4 + k] = o.q[k];
#pragma unroll
  for (int k = 0; k < 3; ++k) w[WORDS + 4 + k] = 0u;
  // pieces that are complete in this lane's hands: all of its aligned ones if it has eight elements (and a left neighbour)
  const bool whole = n >= tail && (off == 0 || lane > 0);
  const bool next_whole = __shfl_down_sync(0xffffffffu, int(whole), 1) != 0 && lane < 31;
  if (whole) {
    const uint32_t back = off == 0 ? 0u : 16u - off;                       // bytes of the neighbour's piece that are not wanted
    if (off == 0) {
#pragma unroll
      for (int k = 0; k < WORDS; ++k) w[k] = w[4 + k];
    } else if constexpr (WORDS == 8) {
      shift_words<8>(w, back >> 2);
    } else {
      shift_words<5>(w, back >> 2);
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = __funnelshift_r(w[k], w[k + 1], (back & 2u) * 8u);
    }
    uint4* to = reinterpret_cast<uint4*>(reinterpret_cast<uintptr_t>(p) - off);
#pragma unroll
    for (int k = 0; k < WORDS / 4; ++k) to[k] = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n && j < tail) p[j] = o.element(j);
  }
  if (off != 0 && !next_whole) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n && j >= tail) p[j] = o.element(j);
  }
}

}  // namespace i8m

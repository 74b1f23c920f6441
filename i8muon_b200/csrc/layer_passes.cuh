// Memory-bound passes of the layers around the stepped matrices: activations to and from eight bits, the
// gradient of a linear layer's pre-activation, sums over rows.
#pragma once
#include "activations.cuh"
#include "eight_bit.cuh"
#include "vectors.cuh"

namespace i8m {

constexpr int EIGHT_THREADS = 256;

__device__ __forceinline__ uint32_t warp_max_u(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }
__device__ __forceinline__ uint32_t magnitude_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// Eight elements of a lane and the group that four neighbouring lanes hold: the exponent byte and the packed codes.
template <int FORMAT>
__device__ __forceinline__ uint32_t quad_exponent(const float (&v)[8]) {
  float most = 0.f;
#pragma unroll
  for (int j = 0; j < 8; j += 2) most = top_of(most, v[j], v[j + 1]);
  uint32_t top = __float_as_uint(most);
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
  return eight_exponent<FORMAT>(top);
}
template <int FORMAT>
__device__ __forceinline__ uint2 encode8(const float (&v)[8], uint32_t byte) {
  const float inverse = eight_inverse(byte);
  return make_uint2(eight_encode4<FORMAT>(v[0], v[1], v[2], v[3], inverse), eight_encode4<FORMAT>(v[4], v[5], v[6], v[7], inverse));
}
template <int FORMAT>
__device__ __forceinline__ void decode8(uint2 codes, uint32_t byte, float (&v)[8]) {
  const float step = eight_step(byte);
  float lo[4], hi[4];
  eight_decode4<FORMAT>(codes.x, step, lo);
  eight_decode4<FORMAT>(codes.y, step, hi);
#pragma unroll
  for (int j = 0; j < 4; ++j) { v[j] = lo[j]; v[4 + j] = hi[j]; }
}

// Widths of whole groups: rows follow one another without gaps, and the tensor is a list of octets (eight elements).  A
// thread takes EIGHT_UNROLL octets, all loaded before the first is used, four neighbouring lanes hold a group.
// Bound by HBM: 2 + 1 + 1/32 bytes per 16-bit element either way.
constexpr int EIGHT_UNROLL = 4;
template <typename E, int FORMAT>
__global__ void __launch_bounds__(EIGHT_THREADS)
eight_quant_octets_kernel(const E* __restrict__ x, uint8_t* __restrict__ codes, uint8_t* __restrict__ exponents, long long octets) {
  pdl_wait();
  const long long first = (long long)blockIdx.x * (EIGHT_THREADS * EIGHT_UNROLL) + threadIdx.x;
  float v[EIGHT_UNROLL][8];
#pragma unroll
  for (int u = 0; u < EIGHT_UNROLL; ++u) {
    const long long i = first + u * EIGHT_THREADS;
    if (i < octets) load8<E>(x + 8 * i, v[u]);
    else for (int j = 0; j < 8; ++j) v[u][j] = 0.f;
  }
#pragma unroll
  for (int u = 0; u < EIGHT_UNROLL; ++u) {
    const long long i = first + u * EIGHT_THREADS;
    const uint32_t byte = quad_exponent<FORMAT>(v[u]);
    if (byte >= EightTop<E, FORMAT>::BYTE) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[u][j] = EightTop<E, FORMAT>::clip(v[u][j]);
    }
    if (i < octets) {
      *reinterpret_cast<uint2*>(codes + 8 * i) = encode8<FORMAT>(v[u], byte);
      if ((i & 3) == 0) exponents[i >> 2] = uint8_t(byte);
    }
  }
}
template <typename E, int FORMAT>
__global__ void __launch_bounds__(EIGHT_THREADS)
eight_restore_octets_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ exponents, E* __restrict__ out,
                            long long octets) {
  pdl_wait();
  const long long first = (long long)blockIdx.x * (EIGHT_THREADS * EIGHT_UNROLL) + threadIdx.x;
  uint2 c[EIGHT_UNROLL];
  uint32_t byte[EIGHT_UNROLL];
#pragma unroll
  for (int u = 0; u < EIGHT_UNROLL; ++u) {
    const long long i = first + u * EIGHT_THREADS;
    if (i < octets) { c[u] = *reinterpret_cast<const uint2*>(codes + 8 * i); byte[u] = exponents[i >> 2]; }
  }
#pragma unroll
  for (int u = 0; u < EIGHT_UNROLL; ++u) {
    const long long i = first + u * EIGHT_THREADS;
    float v[8];
    if (i >= octets) continue;
    decode8<FORMAT>(c[u], byte[u], v);
    store8<E>(out + 8 * i, v);
  }
}

// Any width and alignment: one element per lane, a warp takes EIGHT_SEGMENT groups of a row, four of them in flight.
// blockIdx.y: segment of the row; rows are spread over the warps of blockIdx.x.
constexpr int EIGHT_SEGMENT = 16;
template <typename E, int FORMAT>
__global__ void __launch_bounds__(EIGHT_THREADS)
eight_quant_rows_kernel(const E* __restrict__ x, uint8_t* __restrict__ codes, uint8_t* __restrict__ exponents, long long rows,
                        int width, int groups) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int g0 = blockIdx.y * EIGHT_SEGMENT, g1 = min(groups, g0 + EIGHT_SEGMENT);
  const long long stride = (long long)gridDim.x * (EIGHT_THREADS / 32);
  for (long long row = (long long)blockIdx.x * (EIGHT_THREADS / 32) + (threadIdx.x >> 5); row < rows; row += stride) {
    const E* src = x + row * width + lane;
    uint8_t* dst = codes + row * groups * EIGHT_GROUP + lane;
    for (int g = g0; g < g1; g += EIGHT_UNROLL) {
      float v[EIGHT_UNROLL];
#pragma unroll
      for (int u = 0; u < EIGHT_UNROLL; ++u) {
        const int col = (g + u) * EIGHT_GROUP;
        v[u] = g + u < g1 && col + lane < width ? widen<E>(src[col]) : 0.f;
      }
#pragma unroll
      for (int u = 0; u < EIGHT_UNROLL; ++u) {
        if (g + u >= g1) break;
        const uint32_t byte = eight_exponent<FORMAT>(warp_max_u(magnitude_bits(v[u])));
        if (byte >= EightTop<E, FORMAT>::BYTE) v[u] = EightTop<E, FORMAT>::clip(v[u]);
        dst[(g + u) * EIGHT_GROUP] = eight_encode1<FORMAT>(v[u], eight_inverse(byte));
        if (lane == 0) exponents[row * groups + g + u] = uint8_t(byte);
      }
    }
  }
}
// out: (rows, pitch); elements between width and pitch are written as zero.
template <typename E, int FORMAT>
__global__ void __launch_bounds__(EIGHT_THREADS)
eight_restore_rows_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ exponents, E* __restrict__ out, long long rows,
                          int width, int groups, int pitch) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int g0 = blockIdx.y * EIGHT_SEGMENT, g1 = min(groups, g0 + EIGHT_SEGMENT);
  const long long stride = (long long)gridDim.x * (EIGHT_THREADS / 32);
  for (long long row = (long long)blockIdx.x * (EIGHT_THREADS / 32) + (threadIdx.x >> 5); row < rows; row += stride) {
    const uint8_t* src = codes + row * groups * EIGHT_GROUP + lane;
    const uint8_t* bytes = exponents + row * groups;
    E* dst = out + row * pitch + lane;
    for (int g = g0; g < g1; g += EIGHT_UNROLL) {
      uint8_t c[EIGHT_UNROLL], byte[EIGHT_UNROLL];
#pragma unroll
      for (int u = 0; u < EIGHT_UNROLL; ++u)
        if (g + u < g1) { c[u] = src[(g + u) * EIGHT_GROUP]; byte[u] = bytes[g + u]; }
#pragma unroll
      for (int u = 0; u < EIGHT_UNROLL; ++u) {
        const int col = (g + u) * EIGHT_GROUP;
        if (g + u < g1 && col + lane < pitch)
          dst[col] = round_to<E>(col + lane < width ? eight_decode1<FORMAT>(c[u], eight_step(byte[u])) : 0.f);
      }
    }
  }
}

// ======================================================================= sums over rows
// Sums over rows, in two steps with a fixed order: block (c, p) adds up band p of the rows for 32 columns and leaves
// partials (bands, 2, width); column_fold_kernel adds up the bands.
constexpr int COLUMN_LANES = 8;      // rows that a block reads at a time
__device__ __forceinline__ void store_column_sums(float a, float b, float* partials, int width) {
  __shared__ float sh[2][COLUMN_LANES][32];
  const int c = threadIdx.x & 31, l = threadIdx.x >> 5, col = blockIdx.x * 32 + c;
  sh[0][l][c] = a;
  sh[1][l][c] = b;
  __syncthreads();
  if (l < 2 && col < width) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < COLUMN_LANES; ++i) s += sh[l][i][c];
    partials[(size_t(blockIdx.y) * 2 + l) * width + col] = s;
  }
}
// out0 / out1 (either may be NULL) from partials (bands, 2, width): 32 columns per block, the bands spread over its warps.
constexpr int FOLD_LANES = 16;
template <typename E>
__global__ void __launch_bounds__(32 * FOLD_LANES)
column_fold_kernel(const float* __restrict__ partials, E* __restrict__ out0, E* __restrict__ out1, int width, int bands) {
  __shared__ float sh[FOLD_LANES][32];
  pdl_wait();
  const int c = threadIdx.x & 31, l = threadIdx.x >> 5, col = blockIdx.x * 32 + c, k = blockIdx.y;
  E* out = k == 0 ? out0 : out1;
  if (out == nullptr) return;                 // uniform over the block
  float s = 0.f;
  if (col < width) {
#pragma unroll 4
    for (int p = l; p < bands; p += FOLD_LANES) s += partials[(size_t(p) * 2 + k) * width + col];
  }
  sh[l][c] = s;
  __syncthreads();
  if (l == 0 && col < width) {
#pragma unroll
    for (int i = 1; i < FOLD_LANES; ++i) s += sh[i][c];
    out[col] = round_to<E>(s);
  }
}

// ====================================================================== linear layer
// Rows copied to a pitch that tensor copies can address (a multiple of 16 bytes).
template <typename E>
__global__ void __launch_bounds__(256)
pitch_rows_kernel(const E* __restrict__ src, E* __restrict__ dst, long long rows, int width, int pitch) {
  pdl_wait();
  const int octets = pitch / 8;
  const long long total = rows * octets;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
    const long long row = i / octets;
    const int col = int(i - row * octets) * 8;
    alignas(16) E v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = col + j < width ? src[row * width + col + j] : round_to<E>(0.f);
    *reinterpret_cast<uint4*>(dst + row * pitch + col) = *reinterpret_cast<const uint4*>(v);
  }
}

// What the backward pass knows of the pre-activation.
template <typename E>
struct PreActivation {
  const E* z;               // (rows, z_pitch)
  const uint8_t* codes;     // or eight bits
  const uint8_t* exponents;
  int z_pitch, groups;
};
// dz = dy act'(z) (dz may be NULL) and, where partials is not NULL, its sums over bands of rows for the bias's gradient.
template <typename E, int FORMAT>
__global__ void __launch_bounds__(32 * COLUMN_LANES)
linear_dz_kernel(const E* __restrict__ dy, PreActivation<E> kept, E* __restrict__ dz, float* __restrict__ partials, long long rows,
                 int width, int dz_pitch, long long band, int activation) {
  pdl_wait();
  const int col = blockIdx.x * 32 + (threadIdx.x & 31);
  const long long first = blockIdx.y * band, last = first + band < rows ? first + band : rows;
  float sum = 0.f;
  if (col < width) {
    with_activation(activation, [&](auto act) {
      constexpr int ACT = decltype(act)::value;
      for (long long row = first + (threadIdx.x >> 5); row < last; row += COLUMN_LANES) {
        float v = widen<E>(dy[row * width + col]);
        if constexpr (ACT != ACT_NONE) {
          float z;
          if constexpr (FORMAT >= 0)
            z = eight_decode1<FORMAT>(kept.codes[row * kept.groups * EIGHT_GROUP + col],
                                      eight_step(kept.exponents[row * kept.groups + col / EIGHT_GROUP]));
          else z = widen<E>(kept.z[row * kept.z_pitch + col]);
          v *= lane0(derivative<ACT>(both(z)));
        }
        sum += v;
        if (dz != nullptr) dz[row * dz_pitch + col] = round_to<E>(v);
      }
    });
  }
  if (partials != nullptr) store_column_sums(sum, 0.f, partials, width);
}


// The same where rows of dy, z and dz consist of whole octets on 16 bytes: a lane takes eight columns, a warp 256 of a row, the
// block's warps rows one after the other, DZ_ROWS of them on their way at a time.  Bound by HBM (6 bytes per element, 5 with
// codes); the special functions of an activation come second.
constexpr int DZ_WARPS = 8, DZ_ROWS = 4;
template <typename E, int FORMAT>
__global__ void __launch_bounds__(32 * DZ_WARPS)
linear_dz_octets_kernel(const E* __restrict__ dy, PreActivation<E> kept, E* __restrict__ dz, float* __restrict__ partials,
                        long long rows, int width, long long band, int activation) {
  __shared__ float sums[DZ_WARPS][256];
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, col = (blockIdx.x * 32 + lane) * 8;
  const long long first = blockIdx.y * band, last = first + band < rows ? first + band : rows;
  unsigned long long sum[4] = {0ull, 0ull, 0ull, 0ull};
  if (col < width) {
    with_activation(activation, [&](auto act) {
      constexpr int ACT = decltype(act)::value;
      for (long long row = first + warp; row < last; row += DZ_WARPS * DZ_ROWS) {
        uint4 d[DZ_ROWS], z[DZ_ROWS];
        uint32_t byte[DZ_ROWS];
#pragma unroll
        for (int r = 0; r < DZ_ROWS; ++r) {
          const long long at = row + r * DZ_WARPS;
          if (at >= last) continue;
          d[r] = *reinterpret_cast<const uint4*>(dy + at * width + col);
          if constexpr (ACT == ACT_NONE) continue;
          if constexpr (FORMAT >= 0) {
            const uint2 c = *reinterpret_cast<const uint2*>(kept.codes + at * kept.groups * EIGHT_GROUP + col);
            z[r].x = c.x; z[r].y = c.y;
            byte[r] = kept.exponents[at * kept.groups + col / EIGHT_GROUP];
          } else {
            z[r] = *reinterpret_cast<const uint4*>(kept.z + at * kept.z_pitch + col);
          }
        }
#pragma unroll
        for (int r = 0; r < DZ_ROWS; ++r) {
          const long long at = row + r * DZ_WARPS;
          if (at >= last) continue;
          float v[8], f[8];
          unpack8<E>(d[r], v);
          if constexpr (ACT != ACT_NONE) {
            if constexpr (FORMAT >= 0) decode8<FORMAT>(make_uint2(z[r].x, z[r].y), byte[r], f);
            else unpack8<E>(z[r], f);
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            unsigned long long p = pair(v[2 * k], v[2 * k + 1]);
            if constexpr (ACT != ACT_NONE) p = mul2(p, derivative<ACT>(pair(f[2 * k], f[2 * k + 1])));
            sum[k] = add2(sum[k], p);
            v[2 * k] = lane0(p); v[2 * k + 1] = lane1(p);
          }
          if (dz != nullptr) store8<E>(dz + at * width + col, v);
        }
      }
    });
  }
  if (partials == nullptr) return;
#pragma unroll
  for (int k = 0; k < 4; ++k) { sums[warp][8 * lane + 2 * k] = lane0(sum[k]); sums[warp][8 * lane + 2 * k + 1] = lane1(sum[k]); }
  __syncthreads();
  const int mine = blockIdx.x * 256 + threadIdx.x;
  if (mine < width) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < DZ_WARPS; ++w) s += sums[w][threadIdx.x];
    partials[size_t(blockIdx.y) * 2 * width + mine] = s;
  }
}

}  // namespace i8m

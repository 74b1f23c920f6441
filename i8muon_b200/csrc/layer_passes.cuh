// Memory-bound passes of the layers around the stepped matrices: activations to and from eight bits, the
// gradient of a linear layer's pre-activation, sums over rows.
#pragma once
#include "activations.cuh"
#include "eight_bit.cuh"
#include "octets.cuh"

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

// Any width and alignment: a lane takes an octet, a warp 256 elements of a row at a time.  blockIdx.y: segment of the row;
// rows are spread over the warps of blockIdx.x.
constexpr int EIGHT_SEGMENT = 32;      // groups: four octets per lane
template <typename E, int FORMAT>
__global__ void __launch_bounds__(EIGHT_THREADS)
eight_quant_rows_kernel(const E* __restrict__ x, uint8_t* __restrict__ codes, uint8_t* __restrict__ exponents, long long rows,
                        int width, int groups) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int end = min(groups, int(blockIdx.y + 1) * EIGHT_SEGMENT) * EIGHT_GROUP;
  const long long stride = (long long)gridDim.x * (EIGHT_THREADS / 32);
  for (long long row = (long long)blockIdx.x * (EIGHT_THREADS / 32) + (threadIdx.x >> 5); row < rows; row += stride) {
    Octet<E> o[EIGHT_UNROLL];
#pragma unroll
    for (int u = 0; u < EIGHT_UNROLL; ++u) {
      const int at = int(blockIdx.y) * EIGHT_SEGMENT * EIGHT_GROUP + (u * 32 + lane) * 8;
      load_any<E>(o[u], x + row * width + at, width - at, x, x + rows * width);
    }
#pragma unroll
    for (int u = 0; u < EIGHT_UNROLL; ++u) {
      const int at = int(blockIdx.y) * EIGHT_SEGMENT * EIGHT_GROUP + (u * 32 + lane) * 8;
      float v[8];
#pragma unroll
      for (int k = 0; k < 4; ++k) { v[2 * k] = lane0(o[u].get(k)); v[2 * k + 1] = lane1(o[u].get(k)); }
      const uint32_t byte = quad_exponent<FORMAT>(v);
      if (byte >= EightTop<E, FORMAT>::BYTE) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = EightTop<E, FORMAT>::clip(v[j]);
      }
      if (at < end) {
        *reinterpret_cast<uint2*>(codes + row * groups * EIGHT_GROUP + at) = encode8<FORMAT>(v, byte);
        if ((lane & 3) == 0) exponents[row * groups + at / EIGHT_GROUP] = uint8_t(byte);
      }
    }
  }
}
// out: (rows, pitch); elements between width and pitch are written as zero.  PITCHED: rows of out start on 16 bytes and the
// pitch is whole octets; otherwise the pitch is the width.
template <typename E, int FORMAT, bool PITCHED>
__global__ void __launch_bounds__(EIGHT_THREADS)
eight_restore_rows_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ exponents, E* __restrict__ out, long long rows,
                          int width, int groups, int pitch) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const long long stride = (long long)gridDim.x * (EIGHT_THREADS / 32);
  for (long long row = (long long)blockIdx.x * (EIGHT_THREADS / 32) + (threadIdx.x >> 5); row < rows; row += stride) {
    uint2 c[EIGHT_UNROLL];
    uint32_t byte[EIGHT_UNROLL];
#pragma unroll
    for (int u = 0; u < EIGHT_UNROLL; ++u) {
      const int at = int(blockIdx.y) * EIGHT_SEGMENT * EIGHT_GROUP + (u * 32 + lane) * 8;
      c[u] = make_uint2(0u, 0u);
      byte[u] = 0u;
      if (at < width) {
        c[u] = *reinterpret_cast<const uint2*>(codes + row * groups * EIGHT_GROUP + at);
        byte[u] = exponents[row * groups + at / EIGHT_GROUP];
      }
    }
#pragma unroll
    for (int u = 0; u < EIGHT_UNROLL; ++u) {
      const int at = int(blockIdx.y) * EIGHT_SEGMENT * EIGHT_GROUP + (u * 32 + lane) * 8;
      float v[8];
      decode8<FORMAT>(c[u], byte[u], v);
      Octet<E> o;
      o.pack(v);
      if constexpr (PITCHED) {
        o.cut(width - at);           // a group that reads back as NaN ends with the width
        if (at < pitch) *reinterpret_cast<uint4*>(out + row * pitch + at) = make_uint4(o.q[0], o.q[1], o.q[2], o.q[3]);
      } else {
        store_any<E>(out + row * width + at, min(8, max(0, width - at)), o);
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
// Up to two matrices of the same width in one launch; dst0 or dst1 may be NULL.
template <typename E>
__global__ void __launch_bounds__(256)
pitch_rows_kernel(const E* __restrict__ src0, E* __restrict__ dst0, long long rows0, const E* __restrict__ src1, E* __restrict__ dst1,
                  long long rows1, int width, int pitch) {
  pdl_wait();
  const int octets = pitch / 8;
  const long long first = dst0 != nullptr ? rows0 * octets : 0, total = first + (dst1 != nullptr ? rows1 * octets : 0);
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
    const bool second = i >= first;
    const E* src = second ? src1 : src0;
    E* dst = second ? dst1 : dst0;
    const long long at = second ? i - first : i, row = at / octets;
    const int col = int(at - row * octets) * 8;
    Octet<E> o;
    load_any<E>(o, src + row * width + col, width - col, src, src + (second ? rows1 : rows0) * width);
    *reinterpret_cast<uint4*>(dst + row * pitch + col) = make_uint4(o.q[0], o.q[1], o.q[2], o.q[3]);
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
// dz = dy act'(z) (dz may be NULL) and, where partials is not NULL, its sums over bands of rows for the bias's gradient: partials
// (bands, 2, width), of which the first line of a band is written.  A lane takes eight columns, a warp 256 of a row, the
// block's warps rows one after the other, DZ_ROWS of them on their way at a time (three and three blocks per SM where there is an
// activation: 8192 x 14336 with GELU took 133 us with four rows and two blocks, 126 with two and four, 119 so).  ALIGNED: rows of dy are whole octets on 16
// bytes, as those of z and dz always are; ACTIVE: there is an activation.  Bound by HBM (6 bytes per element, 5 with codes); the special functions of an
// activation come second.
constexpr int DZ_WARPS = 8;
template <typename E, int FORMAT, bool ALIGNED, bool ACTIVE>
__global__ void __launch_bounds__(32 * DZ_WARPS, ACTIVE ? 3 : 4)
linear_dz_kernel(const E* __restrict__ dy, PreActivation<E> kept, E* __restrict__ dz, float* __restrict__ partials, long long rows,
                 int width, int dz_pitch, long long band, int activation) {
  constexpr int DZ_ROWS = ACTIVE ? 3 : 4;
  __shared__ float sums[DZ_WARPS][256];
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, col = (blockIdx.x * 32 + lane) * 8;
  const long long first = blockIdx.y * band, last = first + band < rows ? first + band : rows;
  unsigned long long sum[4] = {0ull, 0ull, 0ull, 0ull};
  if (col < width) {
    auto rows_of = [&](auto act) {
      constexpr int ACT = decltype(act)::value;
      for (long long row = first + warp; row < last; row += DZ_WARPS * DZ_ROWS) {
        Octet<E> d[DZ_ROWS];
        uint4 z[DZ_ROWS];
        [[maybe_unused]] uint32_t byte[DZ_ROWS];
        [[maybe_unused]] uint32_t words[ALIGNED ? 1 : DZ_ROWS][Octet<E>::WORDS + 7];
        // all rows exist and so do all pieces: one decision, and the rows' loads are on their way together
        const long long end_row = row + (DZ_ROWS - 1) * DZ_WARPS;
        [[maybe_unused]] const bool together = !ALIGNED && end_row < last &&
                              load_inside_fits<E>(dy + row * width + col, dy + end_row * width + col, dy, dy + rows * width);
        if constexpr (!ALIGNED) {
          if (together) {
#pragma unroll
            for (int r = 0; r < DZ_ROWS; ++r) load_inside<E>(words[r], dy + (row + r * DZ_WARPS) * width + col);
#pragma unroll
            for (int r = 0; r < DZ_ROWS; ++r) shift_inside<E>(d[r], words[r], dy + (row + r * DZ_WARPS) * width + col, width - col);
          }
        }
#pragma unroll
        for (int r = 0; r < DZ_ROWS; ++r) {
          const long long at = row + r * DZ_WARPS;
          if (at >= last) continue;
          if constexpr (ALIGNED) d[r].load(dy + at * width + col);
          else if (!together) load_any<E>(d[r], dy + at * width + col, width - col, dy, dy + rows * width);
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
          if constexpr (ACT != ACT_NONE) {
            if constexpr (FORMAT >= 0) decode8<FORMAT>(make_uint2(z[r].x, z[r].y), byte[r], f);
            else unpack8<E>(z[r], f);
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            unsigned long long p = d[r].get(k);
            if constexpr (ACT != ACT_NONE) p = mul2(p, derivative<ACT>(pair(f[2 * k], f[2 * k + 1])));
            sum[k] = add2(sum[k], p);
            v[2 * k] = lane0(p); v[2 * k + 1] = lane1(p);
          }
          if (dz != nullptr) store8<E>(dz + at * dz_pitch + col, v);
        }
      }
    };
    if constexpr (ACTIVE) with_activation(activation, rows_of);
    else rows_of(std::integral_constant<int, ACT_NONE>{});
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

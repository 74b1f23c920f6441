// Memory-bound passes of the layers around the stepped matrices: activations to and from eight bits, layer norm.
#pragma once
#include "activations.cuh"
#include "eight_bit.cuh"

namespace i8m {

constexpr int EIGHT_THREADS = 256;

__device__ __forceinline__ uint32_t warp_max_u(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }
__device__ __forceinline__ uint32_t magnitude_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// One warp per group, one element per lane.  codes: (rows, 32 groups), exponents: (rows, groups).
template <typename E, int FORMAT>
__global__ void __launch_bounds__(EIGHT_THREADS)
eight_quant_kernel(const E* __restrict__ x, uint8_t* __restrict__ codes, uint8_t* __restrict__ exponents, long long rows, int width,
                   int groups) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const long long total = rows * groups;
  const long long stride = (long long)gridDim.x * (EIGHT_THREADS / 32);
  for (long long i = (long long)blockIdx.x * (EIGHT_THREADS / 32) + (threadIdx.x >> 5); i < total; i += stride) {
    const long long row = i / groups;
    const int col = int(i - row * groups) * EIGHT_GROUP + lane;
    float v = col < width ? widen<E>(x[row * width + col]) : 0.f;
    const uint32_t byte = eight_exponent<FORMAT>(warp_max_u(magnitude_bits(v)));
    if (byte >= EightTop<E, FORMAT>::BYTE) v = EightTop<E, FORMAT>::clip(v);
    codes[i * EIGHT_GROUP + lane] = eight_encode1<FORMAT>(v, eight_inverse(byte));
    if (lane == 0) exponents[i] = uint8_t(byte);
  }
}
// out: (rows, pitch); elements between width and pitch are written as zero.
template <typename E, int FORMAT>
__global__ void __launch_bounds__(EIGHT_THREADS)
eight_restore_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ exponents, E* __restrict__ out, long long rows,
                     int width, int groups, int pitch) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const long long total = rows * groups;
  const long long stride = (long long)gridDim.x * (EIGHT_THREADS / 32);
  for (long long i = (long long)blockIdx.x * (EIGHT_THREADS / 32) + (threadIdx.x >> 5); i < total; i += stride) {
    const long long row = i / groups;
    const int col = int(i - row * groups) * EIGHT_GROUP + lane;
    const float v = eight_decode1<FORMAT>(codes[i * EIGHT_GROUP + lane], eight_step(exponents[i]));
    if (col < pitch) out[row * pitch + col] = round_to<E>(col < width ? v : 0.f);
  }
}

// ============================================================================ layer norm
//   u = (x - mean) rstd,  rstd = 1 / sqrt(var + eps),  y = u w + b
//   g = dy w,  dx = rstd (g - mean(g) - u mean(g u)),  dw = sum over rows of dy u,  db = sum over rows of dy
// Statistics, u, g and every sum are FP32; the variance is taken around the finished mean.
constexpr int LN_THREADS = 256;

// Sum over the block, the same in every thread.
__device__ __forceinline__ float block_total(float v, float* sh) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  float r = 0.f;
  for (int i = 0; i < int(blockDim.x >> 5); ++i) r += sh[i];
  __syncthreads();
  return r;
}
template <typename E>
__device__ __forceinline__ float or_else(const E* p, int i, float otherwise) { return p != nullptr ? widen<E>(p[i]) : otherwise; }

// One block per row, the row read once per sweep.  FORMAT -1: no codes.
template <typename E, int FORMAT>
__global__ void __launch_bounds__(LN_THREADS)
ln_forward_loop_kernel(const E* __restrict__ x, const E* __restrict__ w, const E* __restrict__ b, E* __restrict__ y,
                       float* __restrict__ mean_out, float* __restrict__ rstd_out, uint8_t* __restrict__ codes,
                       uint8_t* __restrict__ exponents, long long rows, int width, int groups, float eps) {
  __shared__ float sh[LN_THREADS / 32];
  pdl_wait();
  for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
    const E* src = x + row * width;
    float s = 0.f;
    for (int i = threadIdx.x; i < width; i += LN_THREADS) s += widen<E>(src[i]);
    const float mean = block_total(s, sh) / float(width);
    s = 0.f;
    for (int i = threadIdx.x; i < width; i += LN_THREADS) {
      const float d = widen<E>(src[i]) - mean;
      s = fmaf(d, d, s);
    }
    const float rstd = 1.f / sqrtf(block_total(s, sh) / float(width) + eps);
    if (threadIdx.x == 0 && mean_out != nullptr) mean_out[row] = mean;
    if (threadIdx.x == 0 && rstd_out != nullptr) rstd_out[row] = rstd;
    const int end = FORMAT >= 0 ? groups * EIGHT_GROUP : width;    // whole groups: warps stay together
    for (int i = threadIdx.x; i < end; i += LN_THREADS) {
      const float u = i < width ? (widen<E>(src[i]) - mean) * rstd : 0.f;
      if (i < width) y[row * width + i] = round_to<E>(fmaf(u, or_else(w, i, 1.f), or_else(b, i, 0.f)));
      if constexpr (FORMAT >= 0) {
        const uint32_t byte = eight_exponent<FORMAT>(warp_max_u(magnitude_bits(u)));
        codes[row * groups * EIGHT_GROUP + i] = eight_encode1<FORMAT>(u, eight_inverse(byte));
        if ((threadIdx.x & 31) == 0) exponents[row * groups + i / EIGHT_GROUP] = uint8_t(byte);
      }
    }
  }
}

// What the backward pass knows of the normalised rows: x with its rows' statistics, or the codes of u.
template <typename E>
struct LnKept {
  const E* x;
  const float* mean;
  const uint8_t* codes;
  const uint8_t* exponents;
  int groups;
};
template <typename E, int FORMAT>
__device__ __forceinline__ float ln_unit(const LnKept<E>& k, long long row, int width, int i, float mean, float rstd) {
  if constexpr (FORMAT >= 0)
    return eight_decode1<FORMAT>(k.codes[row * k.groups * EIGHT_GROUP + i], eight_step(k.exponents[row * k.groups + i / EIGHT_GROUP]));
  else return (widen<E>(k.x[row * width + i]) - mean) * rstd;
}
template <typename E, int FORMAT>
__global__ void __launch_bounds__(LN_THREADS)
ln_dx_loop_kernel(const E* __restrict__ dy, LnKept<E> kept, const float* __restrict__ rstd_in, const E* __restrict__ w,
                  E* __restrict__ dx, long long rows, int width) {
  __shared__ float sh[LN_THREADS / 32];
  pdl_wait();
  for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
    const float mean = FORMAT >= 0 ? 0.f : kept.mean[row], rstd = rstd_in[row];
    float sg = 0.f, su = 0.f;
    for (int i = threadIdx.x; i < width; i += LN_THREADS) {
      const float g = widen<E>(dy[row * width + i]) * or_else(w, i, 1.f);
      sg += g;
      su = fmaf(g, ln_unit<E, FORMAT>(kept, row, width, i, mean, rstd), su);
    }
    const float mg = block_total(sg, sh) / float(width), mu = block_total(su, sh) / float(width);
    for (int i = threadIdx.x; i < width; i += LN_THREADS) {
      const float g = widen<E>(dy[row * width + i]) * or_else(w, i, 1.f);
      const float u = ln_unit<E, FORMAT>(kept, row, width, i, mean, rstd);
      dx[row * width + i] = round_to<E>((g - mg - u * mu) * rstd);
    }
  }
}

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
template <typename E, int FORMAT>
__global__ void __launch_bounds__(32 * COLUMN_LANES)
ln_columns_kernel(const E* __restrict__ dy, LnKept<E> kept, const float* __restrict__ rstd_in, float* __restrict__ partials,
                  long long rows, int width, long long band) {
  pdl_wait();
  const int col = blockIdx.x * 32 + (threadIdx.x & 31);
  const long long first = blockIdx.y * band, last = first + band < rows ? first + band : rows;
  float dw = 0.f, db = 0.f;
  if (col < width) {
    for (long long row = first + (threadIdx.x >> 5); row < last; row += COLUMN_LANES) {
      const float v = widen<E>(dy[row * width + col]);
      const float mean = FORMAT >= 0 ? 0.f : kept.mean[row];
      dw = fmaf(v, ln_unit<E, FORMAT>(kept, row, width, col, mean, rstd_in[row]), dw);
      db += v;
    }
  }
  store_column_sums(dw, db, partials, width);
}
// out0 / out1 (either may be NULL) from partials (bands, 2, width).
template <typename E>
__global__ void __launch_bounds__(32 * COLUMN_LANES)
column_fold_kernel(const float* __restrict__ partials, E* __restrict__ out0, E* __restrict__ out1, int width, int bands) {
  __shared__ float sh[2][COLUMN_LANES][32];
  pdl_wait();
  const int c = threadIdx.x & 31, l = threadIdx.x >> 5, col = blockIdx.x * 32 + c;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    float s = 0.f;
    if (col < width && (k == 0 ? out0 : out1) != nullptr)
      for (int p = l; p < bands; p += COLUMN_LANES) s += partials[(size_t(p) * 2 + k) * width + col];
    sh[k][l][c] = s;
  }
  __syncthreads();
  E* out = l == 0 ? out0 : out1;
  if (l < 2 && col < width && out != nullptr) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < COLUMN_LANES; ++i) s += sh[l][i][c];
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
          v *= derivative<ACT>(z);
        }
        sum += v;
        if (dz != nullptr) dz[row * dz_pitch + col] = round_to<E>(v);
      }
    });
  }
  if (partials != nullptr) store_column_sums(sum, 0.f, partials, width);
}

}  // namespace i8m

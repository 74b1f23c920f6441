// Layer norm, forward and backward.
#pragma once
#include "layer_passes.cuh"
#include "octets.cuh"

namespace i8m {

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

// ---- rows that fit into registers
// The threads of a row (a warp, or the block) hold V octets each: octet v of thread t is the row's octet v T + t, and a group of
// 32 lies in four neighbouring lanes.  VEC: rows start on 16 bytes (FP32 results on 32) and consist of whole octets; otherwise
// they start anywhere, and what lies behind the width reads as zero.
template <typename E, bool WARP, int V, bool VEC>
struct RowSlice {
  static __device__ __forceinline__ int threads() { return WARP ? 32 : int(blockDim.x); }
  static __device__ __forceinline__ int index(int t, int v) { return 8 * (v * threads() + t); }
  static __device__ __forceinline__ bool inside(int t, int v, int j, int width) { return index(t, v) + (VEC ? 0 : j) < width; }
  // (value, value) for the elements 2 k and 2 k + 1, zero behind the width
  static __device__ __forceinline__ unsigned long long masked(float value, int t, int v, int k, int width) {
    return pair(inside(t, v, 2 * k, width) ? value : 0.f, inside(t, v, 2 * k + 1, width) ? value : 0.f);
  }
  // row of a tensor that ends at `end` (and begins at `begin`)
  static __device__ __forceinline__ void load(const E* row, int width, int t, int v, Octet<E>& o, const E* begin, const E* end) {
    if constexpr (VEC) {
      o.clear();
      if (inside(t, v, 0, width)) o.load(row + index(t, v));
    } else {
      load_any<E>(o, row + index(t, v), width - index(t, v), begin, end);
    }
  }
  static __device__ __forceinline__ void load(const E* vector, int width, int t, int v, Octet<E>& o) {
    load(vector, width, t, v, o, vector, vector + width);
  }
  // all lanes of the warps that hold the row call it
  static __device__ __forceinline__ void store(E* row, int width, int t, int v, const float (&x)[8]) {
    if constexpr (VEC) {
      if (inside(t, v, 0, width)) store8<E>(row + index(t, v), x);
    } else {
      Octet<E> o;
      o.pack(x);
      store_any<E>(row + index(t, v), min(8, max(0, width - index(t, v))), o);
    }
  }
  // Eight bits of x (zero behind the width) to a row of codes and exponents; all lanes of the warps that hold the row call it.
  template <int FORMAT>
  static __device__ __forceinline__ void store_eight(uint8_t* codes, uint8_t* exponents, int groups, int t, int v, const float (&x)[8]) {
    const int at = index(t, v);
    const uint32_t byte = quad_exponent<FORMAT>(x);
    if (at < groups * EIGHT_GROUP) {
      *reinterpret_cast<uint2*>(codes + at) = encode8<FORMAT>(x, byte);
      if ((t & 3) == 0) exponents[at / EIGHT_GROUP] = uint8_t(byte);
    }
  }
};
// Sums over the threads of a row (WARP: one warp, otherwise the block), the same in each: shuffles inside a warp, the warps'
// sums through shared memory.  One barrier: the caller alternates between two buffers.
constexpr int LN_MOST_WARPS = 16;
template <bool WARP>
__device__ __forceinline__ float row_total(float v, float* sh) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if constexpr (!WARP) {
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    v = sh[0];
    for (int i = 1; i < int(blockDim.x >> 5); ++i) v += sh[i];
  }
  return v;
}
// Two sums at once: after the first exchange the lower half of a warp carries one and the upper half the other, and so do
// the warps' sums: sh holds LN_MOST_WARPS pairs, zero where there is no warp (clear_totals).
template <bool WARP>
__device__ __forceinline__ float2 row_total(float2 v, float* sh) {
  const int lane = threadIdx.x & 31, half = lane >> 4;
  float mine = half ? v.y : v.x;
  mine += __shfl_xor_sync(0xffffffffu, half ? v.x : v.y, 16);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  if constexpr (!WARP) {
    if ((lane & 15) == 0) sh[half * LN_MOST_WARPS + (threadIdx.x >> 5)] = mine;
    __syncthreads();
    mine = sh[lane];
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  }
  return make_float2(__shfl_sync(0xffffffffu, mine, 0), __shfl_sync(0xffffffffu, mine, 16));
}
static_assert(LN_MOST_WARPS == 16, "a half warp adds up the warps' sums");
__device__ __forceinline__ void clear_totals(float (&sh)[2][2 * LN_MOST_WARPS]) {
  for (int i = threadIdx.x; i < 4 * LN_MOST_WARPS; i += blockDim.x) (&sh[0][0])[i] = 0.f;
  __syncthreads();
}
// Asynchronous copy of 16 bytes into shared memory; what a thread copies it reads itself, so waiting for its own copies is all.
// FP32 octets are two such pieces of one 32-byte sector, copied one after the other: through L1, which keeps the second.
template <typename E>
__device__ __forceinline__ void copy_async16(uint32_t dst, const void* src) {
  if constexpr (sizeof(E) == 4) asm volatile("cp.async.ca.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_async8(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory"); }

constexpr int LN_WARP_ROWS = 4;                 // rows of a block whose warps hold a row each
constexpr int LN_BLOCK = 512;                   // most threads of a block
// Rows in shared memory, the one that is worked on included: up to four, as far as 208 KB hold `inputs` rows of the widest block
// that many times.
template <typename E, bool WARP, int V>
constexpr int ln_stage_bytes(int inputs) { return (WARP ? 32 * LN_WARP_ROWS : LN_BLOCK) * V * 8 * int(sizeof(E)) * inputs; }
template <typename E, bool WARP, int V, int INPUTS>
constexpr int LN_STAGES = 4 * ln_stage_bytes<E, WARP, V>(INPUTS) <= 208 * 1024 ? 4
                        : 3 * ln_stage_bytes<E, WARP, V>(INPUTS) <= 208 * 1024 ? 3 : 1;

// A row that starts anywhere on its way through shared memory: the aligned 16-byte pieces that hold it, in order, copied by all
// threads of the row and read at the row's offset.  What lies outside the tensor (a first or last piece) is left out.
template <typename E, bool WARP, int V>
struct ShiftedRow {
  static constexpr int PIECES = int(sizeof(E)) / 2;
  static __device__ __forceinline__ int threads() { return WARP ? 32 : int(blockDim.x); }
  static __device__ __forceinline__ uint32_t bytes() { return uint32_t(threads() * V * PIECES + 1) * 16u; }
  static __device__ __forceinline__ void piece(const E* row, int width, int c, const E* begin, const E* end, uint32_t to) {
    const uintptr_t at = (reinterpret_cast<uintptr_t>(row) & ~uintptr_t(15)) + 16u * uint32_t(c);
    if (at >= reinterpret_cast<uintptr_t>(row + width)) return;
    to += 16u * uint32_t(c);
    if (at >= reinterpret_cast<uintptr_t>(begin) && at + 16u <= reinterpret_cast<uintptr_t>(end)) {
      copy_async16<__half>(to, reinterpret_cast<const void*>(at));
    } else {
#pragma unroll
      for (int j = 0; j < 16 / int(sizeof(E)); ++j) {
        const E* e = reinterpret_cast<const E*>(at) + j;
        if (e < begin || e >= end) continue;
        if constexpr (sizeof(E) == 4) asm volatile("st.shared.f32 [%0], %1;" ::"r"(to + 4u * j), "f"(widen<E>(*e)) : "memory");
        else asm volatile("st.shared.u16 [%0], %1;" ::"r"(to + 2u * j), "h"(*reinterpret_cast<const uint16_t*>(e)) : "memory");
      }
    }
  }
  static __device__ __forceinline__ void fetch(const E* row, int width, int t, const E* begin, const E* end, uint32_t to) {
#pragma unroll
    for (int i = 0; i < V * PIECES; ++i) piece(row, width, i * threads() + t, begin, end, to);
    if (t == 0) piece(row, width, V * PIECES * threads(), begin, end, to);
  }
  // octet v of thread t, of which n elements exist, of a row that starts `off` bytes behind its first piece
  static __device__ __forceinline__ void read(uint32_t from, uint32_t off, int t, int v, int n, Octet<E>& o) {
    constexpr int WORDS = Octet<E>::WORDS;
    uint32_t w[WORDS + 7];
#pragma unroll
    for (int k = 0; k < PIECES + 1; ++k) {
      const uint4 q = lds128u(from + uint32_t(((v * threads() + t) * PIECES + k) * 16));
      w[4 * k] = q.x; w[4 * k + 1] = q.y; w[4 * k + 2] = q.z; w[4 * k + 3] = q.w;
    }
    w[WORDS + 4] = w[WORDS + 5] = w[WORDS + 6] = 0u;
    if constexpr (WORDS == 8) {
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
};
template <bool WARP>
__device__ __forceinline__ void row_sync() {
  if constexpr (WARP) __syncwarp();
  else __syncthreads();
}

// Bound by HBM (one read, one write), next to it by issue slots.  So few threads with many elements each (a row's two sums cost
// ten shuffles and a barrier whatever a thread holds), elements widened once, and arithmetic on pairs.  The next rows are on
// their way to shared memory while this one is worked on; rows of whole octets that start on 16 bytes are copied by the
// threads that read them, others (SHIFT) by all and behind a barrier.
template <typename E, bool WARP, int V, bool SHIFT>
__global__ void __launch_bounds__(WARP ? 32 * LN_WARP_ROWS : LN_BLOCK, WARP ? 4 : 1)       // 512 threads per SM
ln_forward_kernel(const E* __restrict__ x, const E* __restrict__ w, const E* __restrict__ b, E* __restrict__ y,
                  float* __restrict__ mean_out, float* __restrict__ rstd_out, uint8_t* __restrict__ codes,
                  uint8_t* __restrict__ exponents, int format, long long rows, int width, int groups, float eps) {
  using Slice = RowSlice<E, WARP, V, !SHIFT>;
  using Shifted = ShiftedRow<E, WARP, V>;
  constexpr int R = WARP ? LN_WARP_ROWS : 1, SLOT = V * 8 * int(sizeof(E)), STAGES = LN_STAGES<E, WARP, V, 1>;
  static_assert(STAGES >= 3, "a row fits three times");
  extern __shared__ __align__(16) uint8_t ln_smem[];
  __shared__ float sh[2][LN_MOST_WARPS];
  pdl_wait();
  const int t = WARP ? threadIdx.x & 31 : threadIdx.x;
  const long long stride = (long long)gridDim.x * R, first = (long long)blockIdx.x * R + (WARP ? threadIdx.x >> 5 : 0);
  // 16-byte pieces of all threads side by side: no bank conflicts; shifted rows: one behind the other
  auto piece = [&](int stage, int k) { return smem_u32(ln_smem) + uint32_t((stage * (SLOT / 16) + k) * blockDim.x + threadIdx.x) * 16u; };
  auto shifted_at = [&](int stage) { return smem_u32(ln_smem) + (uint32_t(WARP ? threadIdx.x >> 5 : 0) * STAGES + uint32_t(stage)) * Shifted::bytes(); };
  auto fetch = [&](long long row, int stage) {
    if (row < rows) {
      if constexpr (SHIFT) {
        Shifted::fetch(x + row * width, width, t, x, x + rows * width, shifted_at(stage));
      } else {
#pragma unroll
        for (int v = 0; v < V; ++v)
          if (Slice::inside(t, v, 0, width)) {
            const E* src = x + row * width + Slice::index(t, v);
#pragma unroll
            for (int k = 0; k < int(sizeof(E)) / 2; ++k)
              copy_async16<E>(piece(stage, v * (int(sizeof(E)) / 2) + k), reinterpret_cast<const uint8_t*>(src) + 16 * k);
          }
      }
    }
    copy_commit();
  };
  Octet<E> wv[V], bv[V];
  const bool scaled = w != nullptr, shifted = b != nullptr;
  const float per_element = 1.f / float(width);
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) fetch(first + s * stride, s);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    if (scaled) Slice::load(w, width, t, v, wv[v]);
    if (shifted) Slice::load(b, width, t, v, bv[v]);
  }
  int stage = 0;
  for (long long row = first; row < rows; row += stride) {
    Octet<E> in[V];
    copy_wait<STAGES - 2>();
    if constexpr (SHIFT) {
      row_sync<WARP>();
      const uint32_t off = uint32_t(reinterpret_cast<uintptr_t>(x + row * width) & 15u);
#pragma unroll
      for (int v = 0; v < V; ++v) Shifted::read(shifted_at(stage), off, t, v, width - Slice::index(t, v), in[v]);
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        in[v].clear();
        if (Slice::inside(t, v, 0, width)) {
#pragma unroll
          for (int k = 0; k < int(sizeof(E)) / 2; ++k) {
            const uint4 q = lds128u(piece(stage, v * (int(sizeof(E)) / 2) + k));
            in[v].q[4 * k] = q.x; in[v].q[4 * k + 1] = q.y; in[v].q[4 * k + 2] = q.z; in[v].q[4 * k + 3] = q.w;
          }
        }
      }
    }
    unsigned long long xs[V][4], sum = 0ull;
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        xs[v][k] = in[v].get(k);
        sum = add2(sum, xs[v][k]);
      }
    const float mean = row_total<WARP>(lane0(sum) + lane1(sum), sh[0]) * per_element;
    // into the stage of the row before this one: its values have been used
    fetch(row + (STAGES - 1) * stride, (stage + STAGES - 1) % STAGES);
    stage = (stage + 1) % STAGES;
    sum = 0ull;
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        xs[v][k] = add2(xs[v][k], Slice::masked(-mean, t, v, k, width));
        sum = fma2(xs[v][k], xs[v][k], sum);
      }
    const float rstd = rsqrtf(fmaf(row_total<WARP>(lane0(sum) + lane1(sum), sh[1]), per_element, eps));
    if (t == 0 && mean_out != nullptr) mean_out[row] = mean;
    if (t == 0 && rstd_out != nullptr) rstd_out[row] = rstd;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float u[8], o[8];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const unsigned long long unit = mul2(xs[v][k], both(rstd));
        unsigned long long out = unit;
        if (scaled && shifted) out = fma2(unit, wv[v].get(k), bv[v].get(k));
        else if (scaled) out = mul2(unit, wv[v].get(k));
        else if (shifted) out = add2(unit, bv[v].get(k));
        u[2 * k] = lane0(unit); u[2 * k + 1] = lane1(unit);
        o[2 * k] = lane0(out); o[2 * k + 1] = lane1(out);
      }
      Slice::store(y + row * width, width, t, v, o);
      if (format == EIGHT_INT8)
        Slice::template store_eight<EIGHT_INT8>(codes + row * groups * EIGHT_GROUP, exponents + row * groups, groups, t, v, u);
      else if (format == EIGHT_E4M3)
        Slice::template store_eight<EIGHT_E4M3>(codes + row * groups * EIGHT_GROUP, exponents + row * groups, groups, t, v, u);
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

// The end of a backward kernel: a block's sums over its rows leave as one line of partials (bands, 2, width).
template <typename E, bool WARP, int V>
__device__ __forceinline__ void store_row_sums(const unsigned long long (&dw)[V][4], const unsigned long long (&db)[V][4], float* partials,
                                               int width) {
  using Slice = RowSlice<E, WARP, V, true>;
  constexpr int R = WARP ? LN_WARP_ROWS : 1;
  const int t = WARP ? threadIdx.x & 31 : threadIdx.x;
  if (partials == nullptr) return;
  float* line = partials + size_t(blockIdx.x) * 2 * width;
  if constexpr (!WARP) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int i = Slice::index(t, v) + j;
        const unsigned long long a = dw[v][j / 2], c = db[v][j / 2];
        if (i < width) { line[i] = j & 1 ? lane1(a) : lane0(a); line[width + i] = j & 1 ? lane1(c) : lane0(c); }
      }
    }
  } else {
    __shared__ float sums[2][32 * V * 8];           // the block's warps add up one after the other
    for (int turn = 0; turn < R; ++turn) {
      if (int(threadIdx.x >> 5) == turn) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int i = Slice::index(t, v) + j;
            const unsigned long long a = dw[v][j / 2], c = db[v][j / 2];
            sums[0][i] = (turn ? sums[0][i] : 0.f) + (j & 1 ? lane1(a) : lane0(a));
            sums[1][i] = (turn ? sums[1][i] : 0.f) + (j & 1 ? lane1(c) : lane0(c));
          }
        }
      }
      __syncthreads();
    }
    for (int i = threadIdx.x; i < width; i += 32 * LN_WARP_ROWS) { line[i] = sums[0][i]; line[width + i] = sums[1][i]; }
  }
}

// Rows in registers: one read of dy and of what was kept serves dx and both sums over rows.  A thread keeps the same columns
// for all rows of its block (blockIdx.x, blockIdx.x + gridDim.x, ...) and adds them up in registers.
//
// Bound by issue slots and HBM alike (at 16384 rows of 4096 BF16 a first version with
// scalar arithmetic issued 34 instructions per 32 elements' worth of work, 2.6 a cycle).  Hence: arithmetic on pairs, two sums
// for the price of one exchange, pointers that advance instead of row * width, and a ring of rows in shared memory that each
// thread fills for itself with asynchronous copies, 16-byte pieces of all threads side by side (with a thread's pieces
// together, 272 bytes from its neighbour's, a pass took 109 us instead of 81).  Twice the threads with one octet each, and so 32
// warps per SM instead of 16, took 102 us: the exchanges of the row's sums are per warp.
// SHIFT: rows that start anywhere, their pieces copied by all threads of the row and read behind a barrier.
// V <= 2 keeps u and g in registers between the two sweeps; V = 4 (rows above 8192) reads them again from shared memory.
template <typename E, bool WARP, int V, int FORMAT, bool SHIFT>
__global__ void __launch_bounds__(WARP ? 32 * LN_WARP_ROWS : LN_BLOCK)
ln_backward_kernel(const E* __restrict__ dy, LnKept<E> kept, const float* __restrict__ rstd_in, const E* __restrict__ w,
                   E* __restrict__ dx, float* __restrict__ partials, long long rows, int width) {
  constexpr int R = WARP ? LN_WARP_ROWS : 1, PIECES = int(sizeof(E)) / 2;   // 16-byte pieces of an octet
  constexpr int STAGES = LN_STAGES<E, WARP, V, 2>;                          // 1: a row is fetched when its turn comes
  constexpr int STAGE_PIECES = 2 * V * PIECES;
  constexpr bool HOLD = V <= 2;
  using Shifted = ShiftedRow<E, WARP, V>;
  extern __shared__ __align__(16) uint8_t ln_smem[];
  __shared__ float sh[2][2 * LN_MOST_WARPS];
  clear_totals(sh);
  pdl_wait();
  const int t = WARP ? threadIdx.x & 31 : threadIdx.x, threads = WARP ? 32 : int(blockDim.x);
  const long long stride = (long long)gridDim.x * R, first = (long long)blockIdx.x * R + (WARP ? threadIdx.x >> 5 : 0);
  const long long count = first < rows ? (rows - first + stride - 1) / stride : 0;
  // stages are `stage_bytes` apart from `mine` on: pieces of all threads side by side, or (SHIFT) a row's two inputs in order
  const uint32_t apart = uint32_t(blockDim.x) * 16u, stage_bytes = SHIFT ? 2u * Shifted::bytes() : uint32_t(STAGE_PIECES) * apart;
  const uint32_t mine = smem_u32(ln_smem) + (SHIFT ? uint32_t(WARP ? threadIdx.x >> 5 : 0) * uint32_t(STAGES) * stage_bytes : uint32_t(threadIdx.x) * 16u);
  bool inside[V];
#pragma unroll
  for (int v = 0; v < V; ++v) inside[v] = 8 * (v * threads + t) < width;

  // what is fetched next: pointers to this thread's first octet of the row, and how many rows are left to fetch
  const long long step = stride * width;
  const E* next_dy = dy + first * width + (SHIFT ? 0 : 8 * t);
  const E* next_x = FORMAT < 0 ? kept.x + first * width + (SHIFT ? 0 : 8 * t) : nullptr;
  // bytes by which this row and its kept row start behind a piece, and what they gain from row to row
  uint32_t off_dy = uint32_t(reinterpret_cast<uintptr_t>(next_dy) & 15u), off_x = FORMAT < 0 ? uint32_t(reinterpret_cast<uintptr_t>(next_x) & 15u) : 0u;
  const uint32_t off_step = uint32_t((unsigned long long)step * sizeof(E)) & 15u;
  const long long code_step = stride * kept.groups * EIGHT_GROUP, byte_step = stride * kept.groups;
  const uint8_t* next_codes = FORMAT >= 0 ? kept.codes + first * kept.groups * EIGHT_GROUP + 8 * t : nullptr;
  long long to_fetch = count;
  auto fetch = [&](uint32_t at) {
    if (to_fetch > 0) {
      if constexpr (SHIFT) {
        Shifted::fetch(next_dy, width, t, dy, dy + rows * width, at);
        if constexpr (FORMAT < 0) Shifted::fetch(next_x, width, t, kept.x, kept.x + rows * width, at + Shifted::bytes());
      }
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (!inside[v]) continue;
        if constexpr (SHIFT) {
          if (FORMAT >= 0) copy_async8(at + Shifted::bytes() + uint32_t(v * threads + t) * 8u, next_codes + 8 * v * threads);
        } else {
#pragma unroll
          for (int k = 0; k < PIECES; ++k) {
            copy_async16<E>(at + uint32_t(v * PIECES + k) * apart, reinterpret_cast<const uint8_t*>(next_dy + 8 * v * threads) + 16 * k);
            if (FORMAT < 0) copy_async16<E>(at + uint32_t((V + v) * PIECES + k) * apart, reinterpret_cast<const uint8_t*>(next_x + 8 * v * threads) + 16 * k);
          }
          if (FORMAT >= 0) copy_async8(at + uint32_t((V + v) * PIECES) * apart, next_codes + 8 * v * threads);
        }
      }
      next_dy += step;
      if (FORMAT < 0) next_x += step;
      else next_codes += code_step;
      --to_fetch;
    }
    copy_commit();
  };
  // a row's statistics and exponent bytes, one row ahead in registers
  const float *rstd_at = rstd_in + first, *mean_at = FORMAT < 0 ? kept.mean + first : nullptr;
  const uint8_t* bytes_at = FORMAT >= 0 ? kept.exponents + first * kept.groups + t / 4 : nullptr;
  float next_mean = 0.f, next_rstd = 0.f;
  uint32_t next_byte[V];
  auto fetch_small = [&]() {
    next_rstd = *rstd_at;
    rstd_at += stride;
    if (FORMAT < 0) { next_mean = *mean_at; mean_at += stride; }
    else {
#pragma unroll
      for (int v = 0; v < V; ++v) next_byte[v] = inside[v] ? bytes_at[v * threads / 4] : 0u;
      bytes_at += byte_step;
    }
  };

  unsigned long long dw[V][4], db[V][4];
#pragma unroll
  for (int v = 0; v < V; ++v)
#pragma unroll
    for (int k = 0; k < 4; ++k) dw[v][k] = db[v][k] = 0ull;
  const float per_element = 1.f / float(width);
  const bool scaled = w != nullptr;
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) fetch(mine + uint32_t(s) * stage_bytes);
  Octet<E> wv[V];
  auto load_w = [&](int v) {
    wv[v].clear();
    if constexpr (SHIFT) load_any<E>(wv[v], w + 8 * (v * threads + t), width - 8 * (v * threads + t), w, w + width);
    else if (inside[v]) wv[v].load(w + 8 * (v * threads + t));
  };
  if (HOLD && scaled) {
#pragma unroll
    for (int v = 0; v < V; ++v) load_w(v);
  }
  if (count > 0) fetch_small();
  uint32_t at = 0, refill = uint32_t(STAGES - 1) * stage_bytes;    // offsets of this row's stage and of the free one
  E* out = dx != nullptr ? dx + first * width + 8 * t : nullptr;
  int turn = 0;
  for (long long i = 0; i < count; ++i) {
    if (STAGES == 1) {
      if (SHIFT) row_sync<WARP>();              // the only stage has been read by all
      fetch(mine);
    }
    copy_wait<STAGES == 1 ? 0 : STAGES - 2>();
    if (SHIFT) row_sync<WARP>();
    const float mean = next_mean, rstd = next_rstd;
    uint32_t byte[V];
#pragma unroll
    for (int v = 0; v < V; ++v) byte[v] = FORMAT >= 0 ? next_byte[v] : 0u;
    if (i + 1 < count) fetch_small();
    auto octet = [&](int v, Octet<E>& d, unsigned long long (&u)[4], unsigned long long (&g)[4]) {
      Octet<E> raw;
      d.clear();
      raw.clear();
      if constexpr (SHIFT) {
        const int n = width - 8 * (v * threads + t);
        Shifted::read(mine + at, off_dy, t, v, n, d);
        if constexpr (FORMAT < 0) {
          Shifted::read(mine + at + Shifted::bytes(), off_x, t, v, n, raw);
        } else if (inside[v]) {
          const uint32_t c = mine + at + Shifted::bytes() + uint32_t(v * threads + t) * 8u;
          raw.q[0] = lds32u(c); raw.q[1] = lds32u(c + 4u);
        }
      } else if (inside[v]) {
#pragma unroll
        for (int k = 0; k < PIECES; ++k) {
          const uint4 q = lds128u(mine + at + uint32_t(v * PIECES + k) * apart);
          d.q[4 * k] = q.x; d.q[4 * k + 1] = q.y; d.q[4 * k + 2] = q.z; d.q[4 * k + 3] = q.w;
          if (FORMAT >= 0 && k > 0) continue;
          const uint4 r = lds128u(mine + at + uint32_t((V + v) * PIECES + k) * apart);
          raw.q[4 * k] = r.x; raw.q[4 * k + 1] = r.y; raw.q[4 * k + 2] = r.z; raw.q[4 * k + 3] = r.w;
        }
      }
      if constexpr (FORMAT < 0) {             // behind the width dy is zero
#pragma unroll
        for (int k = 0; k < 4; ++k) u[k] = mul2(add2(raw.get(k), both(-mean)), both(rstd));
      } else {
        float f[8];
        decode8<FORMAT>(make_uint2(raw.q[0], raw.q[1]), byte[v], f);
#pragma unroll
        for (int k = 0; k < 4; ++k) u[k] = pair(f[2 * k], f[2 * k + 1]);
      }
      if (!HOLD && scaled) load_w(v);
#pragma unroll
      for (int k = 0; k < 4; ++k) g[k] = scaled ? mul2(d.get(k), wv[v].get(k)) : d.get(k);
    };
    unsigned long long sg = 0ull, su = 0ull, us[HOLD ? V : 1][4], gs[HOLD ? V : 1][4];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      Octet<E> d;
      unsigned long long (&u)[4] = us[HOLD ? v : 0];
      unsigned long long (&g)[4] = gs[HOLD ? v : 0];
      octet(v, d, u, g);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        dw[v][k] = fma2(d.get(k), u[k], dw[v][k]);
        db[v][k] = add2(db[v][k], d.get(k));
        sg = add2(sg, g[k]);
        su = fma2(g[k], u[k], su);
      }
    }
    if (dx != nullptr) {                          // uniform over the grid
      const float2 s = row_total<WARP>(make_float2(lane0(sg) + lane1(sg), lane0(su) + lane1(su)), sh[turn]);
      turn ^= 1;
      const unsigned long long mg = both(-s.x * per_element), mu = both(-s.y * per_element);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        Octet<E> d;
        float o[8];
        unsigned long long (&u)[4] = us[HOLD ? v : 0];
        unsigned long long (&g)[4] = gs[HOLD ? v : 0];
        if constexpr (!HOLD) octet(v, d, u, g);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const unsigned long long q = mul2(fma2(mu, u[k], add2(g[k], mg)), both(rstd));
          o[2 * k] = lane0(q); o[2 * k + 1] = lane1(q);
        }
        if constexpr (SHIFT) {
          Octet<E> packed;
          packed.pack(o);
          store_any<E>(out + 8 * v * threads, min(8, max(0, width - 8 * (v * threads + t))), packed);
        } else if (inside[v]) {
          store8<E>(out + 8 * v * threads, o);
        }
      }
      out += step;
    }
    // the free stage held the row before this one, whose values have been used
    if (STAGES > 1) {
      fetch(mine + refill);
      refill = at;
      at += stage_bytes;
      if (at == uint32_t(STAGES) * stage_bytes) at = 0;
    }
    off_dy = (off_dy + off_step) & 15u;
    off_x = (off_x + off_step) & 15u;
  }
  store_row_sums<E, WARP, V>(dw, db, partials, width);
}

// ---- wider rows: the sums over rows apart, see store_column_sums
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

}  // namespace i8m

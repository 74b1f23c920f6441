// Epilogue of a linear layer's products (FP16 / BF16 operands, FP32 accumulation):
//   z = acc + bias,  y = act(z) + residual
// in FP32, rounded once.  In training the pre-activation z leaves beside y for the backward pass, rounded to the operand
// type or in eight bits: a thread holds 32 columns of one row, which is a group of that format, so its exponent needs no
// exchange.  The two backward products run through the same epilogue with nothing but y.
//
// What bounds it is instruction issue, not the stores: without them a product with K = 64 took 65 us instead of 68, without
// anything behind the accumulator 35.  Hence one switch over the activations around a warp's blocks, blocks that leave
// as tensor copies (one request of one lane, clipped by the copy engine, instead of four loads and stores per lane with
// their predicates), and a residual that is on its way to L2 while the unit before it is finished.
#pragma once
#include "activations.cuh"
#include "eight_bit.cuh"

namespace i8m {

struct LinearArgs {
  void* y;                 // (lm, ln) in E
  const void* bias;        // [ln] or NULL
  const void* residual;    // (lm, ln) or NULL
  void* z;                 // kept pre-activation: (lm, z_pitch) in E, z_pitch a multiple of 8, or NULL
  uint8_t* codes;          // or in eight bits: (lm, 32 groups), (lm, groups), or NULL
  uint8_t* exponents;
  int z_pitch, groups, format, activation;
  int y_blocks;            // rows of y start on 16 bytes: blocks leave as tensor copies
  float* parts;            // a sum cut into `part_count` runs of K blocks: (part_count, lm, z_pitch) FP32 instead of y, or NULL
  int part_count;
};

__device__ __forceinline__ bool on_16_bytes(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Block of 16-bit values whose rows start anywhere into the patch: one element per lane, a row per request.
__device__ __forceinline__ void load_block_elements16(const WarpPatch& wp, const uint16_t* src, size_t pitch, int rows, int cols) {
  const uint32_t within = uint32_t((wp.lane & 7) * 2);
#pragma unroll 8
  for (int r = 0; r < 32; ++r) {
    const uint16_t v = r < rows && wp.lane < cols ? src[size_t(r) * pitch + wp.lane] : uint16_t(0);
    asm volatile("st.shared.u16 [%0], %1;" ::"r"(wp.piece(r, wp.lane >> 3) + within), "h"(v) : "memory");
  }
}

template <typename E>
__device__ __forceinline__ void pack_row(const unsigned long long (&v)[16], uint32_t (&p)[16]) {
#pragma unroll
  for (int k = 0; k < 16; ++k) p[k] = pack2<E>(lane0(v[k]), lane1(v[k]));
}
template <typename E>
__device__ __forceinline__ unsigned long long widen2(uint32_t v) {
  const float2 f = unpack2<E>(v);
  return pair(f.x, f.y);
}

// Eight bits of one group held by one thread, stored as two 16-byte vectors and a byte.
template <int FORMAT>
__device__ __forceinline__ void store_group(const unsigned long long (&z)[16], uint8_t* codes, uint8_t* exponent) {
  float top = 0.f;
#pragma unroll
  for (int k = 0; k < 16; ++k) top = top_of(top, lane0(z[k]), lane1(z[k]));
  const uint32_t byte = eight_exponent<FORMAT>(__float_as_uint(top));
  const float inverse = eight_inverse(byte);
  uint32_t c[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) c[j] = eight_encode4<FORMAT>(lane0(z[2 * j]), lane1(z[2 * j]), lane0(z[2 * j + 1]), lane1(z[2 * j + 1]), inverse);
  reinterpret_cast<uint4*>(codes)[0] = make_uint4(c[0], c[1], c[2], c[3]);
  reinterpret_cast<uint4*>(codes)[1] = make_uint4(c[4], c[5], c[6], c[7]);
  *exponent = uint8_t(byte);
}

template <typename E>
struct EpiLinear {
  static constexpr int KIND = KIND_F16;
  using Elem = E;
  static constexpr int PARTS = 1;
  static constexpr bool BLOCKQ = false;
  static constexpr int PROMOTE_KB = 0;
  static constexpr uint32_t FMT = std::is_same<E, __nv_bfloat16>::value ? 1u : 0u;
  static constexpr uint32_t IDESC = make_idesc(1u, FMT, FMT, TILE, TILE);
  using Args = LinearArgs;

  // A 32 x 32 block held one row per lane leaves as one tensor copy (a box of 32 rows of 64 bytes, swizzled within 512 bytes),
  // clipped to the tensor.  The copy reads the patch after this returns: patch_free before its next use.
  static __device__ __forceinline__ void patch_free(const WarpPatch& wp) {
    if (wp.lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    __syncwarp();
  }
  static __device__ __forceinline__ void store_block(const WarpPatch& wp, const CUtensorMap* map, int col, int row, const uint32_t (&p)[16]) {
    patch_free(wp);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      sts128u(wp.base + uint32_t(wp.lane * 64 + ((i ^ (wp.lane >> 1)) & 3) * 16), make_uint4(p[4 * i], p[4 * i + 1], p[4 * i + 2], p[4 * i + 3]));
    fence_proxy_async();
    __syncwarp();
    if (wp.lane == 0) {
      asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(reinterpret_cast<uint64_t>(map)),
                   "r"(wp.base), "r"(col), "r"(row), "r"(0)
                   : "memory");
      asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    }
  }

  // Brings the residual's row `row` of a warp's 64 columns from `col` on into L2: called a unit ahead of its use.
  static __device__ __forceinline__ void expect_residual(const GemmGeom& g, const Args& a, int row, int col) {
    if (a.residual == nullptr || row >= g.lm || col >= g.ln) return;
    const E* r = static_cast<const E*>(a.residual) + size_t(row) * g.ln;
    asm volatile("prefetch.global.L2 [%0];" ::"l"(r + col));
    asm volatile("prefetch.global.L2 [%0];" ::"l"(r + min(col + 63, g.ln - 1)));
  }

  // This warp's blocks as FP32 rows of one part of the sum.
  template <class Acc>
  static __device__ __forceinline__ void park(const GemmGeom& g, const Args& a, int part, const TileCtx& t, const Acc& acc) {
#pragma unroll 1
    for (int c = t.c_begin; c < t.c_end; ++c) {
      const int colb = t.col0 + c * 32;
      if (colb >= g.ln) continue;                                  // uniform over the warp
      uint32_t v[32];
      acc.load(c, v);
      float* line = a.parts + (size_t(part) * g.lm + t.row) * a.z_pitch + colb;
      if (t.row >= g.lm) continue;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (colb + 8 * q >= a.z_pitch) continue;
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = __uint_as_float(v[8 * q + j]);
        store8<float>(line + 8 * q, f);
      }
    }
  }

  // This warp's blocks of the tile.
  template <int ACT, class Acc>
  static __device__ __forceinline__ void blocks(const GemmGeom& g, const Args& a, const CUtensorMap* map_y, const CUtensorMap* map_z,
                                                const TileCtx& t, const Acc& acc) {
    const WarpPatch wp{smem_u32(t.wsm), t.lane};
    const int wrow0 = t.row0 + 32 * t.q;
    const bool residual_vectors = a.residual != nullptr && (g.ln & 7) == 0 && on_16_bytes(a.residual);
#pragma unroll 1
    for (int c = t.c_begin; c < t.c_end; ++c) {
      const int colb = t.col0 + c * 32;
      if (colb >= g.ln || wrow0 >= g.lm) continue;               // uniform over the warp
      const BlockClip clip{g.lm - wrow0, g.ln - colb};
      uint32_t v[32];
      acc.load(c, v);
      unsigned long long z[16];
#pragma unroll
      for (int k = 0; k < 16; ++k) z[k] = pack2(v[2 * k], v[2 * k + 1]);
      if (a.bias != nullptr) {
        const E* bias = static_cast<const E*>(a.bias) + colb;
        if (clip.cols >= 32 && on_16_bytes(bias)) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const uint4 w = __ldg(reinterpret_cast<const uint4*>(bias) + q);
            const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) z[4 * q + k] = add2(z[4 * q + k], widen2<E>(words[k]));
          }
        } else {
#pragma unroll
          for (int k = 0; k < 16; ++k)
            z[k] = add2(z[k], pair(2 * k < clip.cols ? widen<E>(bias[2 * k]) : 0.f, 2 * k + 1 < clip.cols ? widen<E>(bias[2 * k + 1]) : 0.f));
        }
      }
      uint32_t p[16];
      if (a.z != nullptr) {
        pack_row<E>(z, p);
        store_block(wp, map_z, colb, wrow0, p);
      }
      if (a.codes != nullptr && t.row < g.lm) {
        const size_t group = size_t(t.row) * a.groups + (colb >> 5);
        if (a.format == EIGHT_INT8) store_group<EIGHT_INT8>(z, a.codes + group * 32, a.exponents + group);
        else store_group<EIGHT_E4M3>(z, a.codes + group * 32, a.exponents + group);
      }
#pragma unroll
      for (int k = 0; k < 16; ++k) z[k] = activate<ACT>(z[k]);
      if (a.residual != nullptr) {
        patch_free(wp);
        const E* r = static_cast<const E*>(a.residual) + size_t(wrow0) * g.ln + colb;
        if (residual_vectors) load_block_rows(wp, reinterpret_cast<const uint8_t*>(r), size_t(g.ln) * 2, clip.rows, clip.cols * 2);
        else load_block_elements16(wp, reinterpret_cast<const uint16_t*>(r), size_t(g.ln), clip.rows, clip.cols);
        __syncwarp();
        wp.read_own_row(p);
        __syncwarp();
#pragma unroll
        for (int k = 0; k < 16; ++k) z[k] = add2(z[k], widen2<E>(p[k]));
      }
      pack_row<E>(z, p);
      if (a.y_blocks) {
        store_block(wp, map_y, colb, wrow0, p);
      } else {
        patch_free(wp);
        wp.write_own_row(p);
        __syncwarp();
        store_block_elements16(wp, reinterpret_cast<uint16_t*>(a.y) + size_t(wrow0) * g.ln + colb, size_t(g.ln), clip.rows, clip.cols);
        __syncwarp();
      }
    }
  }
  template <class Acc>
  static __device__ __forceinline__ void run(const GemmGeom& g, const Args& a, const CUtensorMap* map_y, const CUtensorMap* map_z,
                                             const TileCtx& t, const Acc& acc) {
    with_activation(a.activation, [&](auto act) { blocks<decltype(act)::value>(g, a, map_y, map_z, t, acc); });
  }
};

}  // namespace i8m

// Products of a linear layer with few output tiles, split along K over a cluster of CTAs:  out[c][f] = sum_k B[c][k] A[f][k].
//
// A CTA tile has 128 features f (the contiguous side of the output, on the accumulator's lanes) and BN columns c (rows of the
// output: tokens, or a weight's rows): a product over one to 16 tokens multiplies 16 columns instead of 128.  The K blocks
// of a tile are cut into one run per CTA of a cluster of 1, 2, 4 or 8.  Each CTA parks its FP32 partial tile in shared memory;
// after a cluster barrier the CTAs share out the tile's columns, and a warp finishes a column: it adds up the partial sums
// in the order of the CTAs (read over distributed shared memory) and runs the fused epilogue, four features per lane, so
// that rows leave as 256 contiguous bytes.  Nothing is summed by atomics: the same call gives the same bits.
//
//   warp 0       TMA producer          warp 1       tcgen05.mma issuer (M = 128, N = BN, one accumulator)
//   warps 4..7   read the accumulator and park it       all warps   sum and epilogue
//
// What bounds it: reading A.  One token through 4096 x 4096 BF16 weights reads 33.6 MB; units of 256 columns are 16 for
// that and took 25 us, 32 tiles x 4 CTAs here 10.4, of which 4.5 are a launch's start, barriers and end.  Two CTAs fit on an SM (about 100 KB each), so that one streams while
// the other starts or ends.
#pragma once
#include "epi_linear.cuh"
#include "gemm_fp32_cluster.cuh"

namespace i8m {

constexpr int LSP_THREADS = 256;
constexpr int LSP_PARK_PITCH = TILE + 4;      // floats of a parked column
template <int BN>
struct LinearSplitShape {
  static constexpr int STAGE_BYTES = TILE_BYTES + BN * 128;
  static constexpr int STAGES = BN <= 32 ? 5 : BN == 64 ? 4 : 3;
  static constexpr size_t SMEM = size_t(STAGES) * STAGE_BYTES + sizeof(Ctrl) + 1024;
  static_assert(BN * LSP_PARK_PITCH * 4 <= STAGES * STAGE_BYTES, "the parked tile lies over the ring");
  static_assert(2 * (SMEM + 1024) <= 228 * 1024, "two CTAs per SM");
};

struct LinearSplitGeom {
  int features, columns, num_kb;
  int tiles_f, split;
  int starve;               // test hook: the producer issues nothing
  unsigned* status;
};

// Four features of one column: bias, what is kept, activation, residual, store.  `valid` of the four exist; VEC: all do, and
// every vector involved lies on 8 bytes.
template <typename E>
struct QuadIo {
  static __device__ __forceinline__ void load(const E* p, bool vec, int valid, float (&v)[4]) {
    if (vec) {
      const uint2 w = *reinterpret_cast<const uint2*>(p);
      const float2 a = unpack2<E>(w.x), b = unpack2<E>(w.y);
      v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = j < valid ? widen<E>(p[j]) : 0.f;
    }
  }
  static __device__ __forceinline__ void store(E* p, bool vec, int valid, const float (&v)[4]) {
    if (vec) {
      *reinterpret_cast<uint2*>(p) = make_uint2(pack2<E>(v[0], v[1]), pack2<E>(v[2], v[3]));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < valid) p[j] = round_to<E>(v[j]);
    }
  }
};
__device__ __forceinline__ bool on_8_bytes(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 7u) == 0; }

template <typename E, int FORMAT>
__device__ __forceinline__ void store_quad_group(const float (&z)[4], uint8_t* codes, uint8_t* exponent, bool there, int lane) {
  uint32_t top = __float_as_uint(top_of(top_of(0.f, z[0], z[1]), z[2], z[3]));
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  const uint32_t byte = eight_exponent<FORMAT>(top);
  if (!there) return;
  *reinterpret_cast<uint32_t*>(codes) = eight_encode4<FORMAT>(z[0], z[1], z[2], z[3], eight_inverse(byte));
  if ((lane & 7) == 0) *exponent = uint8_t(byte);
}

// Column `c` of the output, this lane's features f .. f + 3 with sums z.  All lanes of the warp call it.
template <typename E>
__device__ __forceinline__ void linear_column(const LinearArgs& a, const LinearSplitGeom& g, int c, int f, float (&z)[4], int lane) {
  const int valid = g.features - f;
  const bool there = valid > 0, four = valid >= 4 && (g.features & 3) == 0;
  float v[4];
  if (a.bias != nullptr && there) {
    const E* p = static_cast<const E*>(a.bias) + f;
    QuadIo<E>::load(p, four && on_8_bytes(p), valid, v);
#pragma unroll
    for (int j = 0; j < 4; ++j) z[j] += v[j];
  }
  if (a.z != nullptr && there)
    QuadIo<E>::store(static_cast<E*>(a.z) + size_t(c) * a.z_pitch + f, true, 4, z);    // the pitch is a multiple of 8
  if (a.codes != nullptr) {
    const size_t row = size_t(c) * a.groups;
    const bool group = f < a.groups * 32;
    if (a.format == EIGHT_INT8) store_quad_group<E, EIGHT_INT8>(z, a.codes + row * 32 + f, a.exponents + row + f / 32, group, lane);
    else store_quad_group<E, EIGHT_E4M3>(z, a.codes + row * 32 + f, a.exponents + row + f / 32, group, lane);
  }
  if (!there) return;
  with_activation(a.activation, [&](auto act) {
    const unsigned long long y0 = activate<decltype(act)::value>(pair(z[0], z[1])), y1 = activate<decltype(act)::value>(pair(z[2], z[3]));
    z[0] = lane0(y0); z[1] = lane1(y0); z[2] = lane0(y1); z[3] = lane1(y1);
  });
  const size_t at = size_t(c) * g.features + f;
  if (a.residual != nullptr) {
    const E* p = static_cast<const E*>(a.residual) + at;
    QuadIo<E>::load(p, four && on_8_bytes(p), valid, v);
#pragma unroll
    for (int j = 0; j < 4; ++j) z[j] += v[j];
  }
  E* y = static_cast<E*>(a.y) + at;
  QuadIo<E>::store(y, four && on_8_bytes(y), valid, z);
}

template <typename E, int BN, int A_MN, int B_MN>
__global__ void __launch_bounds__(LSP_THREADS, 2)
linear_split_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, LinearSplitGeom g,
                    LinearArgs args) {
  using Shape = LinearSplitShape<BN>;
  using Tiles = OperandTiles<E, A_MN, B_MN>;
  constexpr int STAGES = Shape::STAGES, STAGE_BYTES = Shape::STAGE_BYTES;
  constexpr int TMEM_COLS = BN < 32 ? 32 : BN;
  constexpr uint32_t FMT = std::is_same<E, __nv_bfloat16>::value ? 1u : 0u;
  constexpr uint32_t IDESC = make_idesc(1u, FMT, FMT, TILE, BN) | Tiles::IDESC_BITS;
  static_assert(!B_MN || BN >= 64, "an MN-major box is 64 elements wide");

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Ctrl* ctrl = reinterpret_cast<Ctrl*>(smem + STAGES * STAGE_BYTES);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = g.split, rank = int(blockIdx.x) % split, tile = int(blockIdx.x) / split;
  const int f0 = (tile % g.tiles_f) * TILE, c0 = (tile / g.tiles_f) * BN;
  const int kb0 = int((long long)g.num_kb * rank / split), kb1 = int((long long)g.num_kb * (rank + 1) / split);

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(smem_u32(&ctrl->full[s]), 1);
      mbar_init(smem_u32(&ctrl->empty[s]), 1);
    }
    mbar_init(smem_u32(&ctrl->acc_full[0]), 1);
    ctrl->abort = 0;
    fence_mbar_init();
    tma_prefetch_desc(&map_a);
    tma_prefetch_desc(&map_b);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&ctrl->tmem_base), TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait();
  const uint32_t tmem_base = ctrl->tmem_base, smem_base = smem_u32(smem);
  volatile uint32_t* abort_flag = &ctrl->abort;

  if (warp == 0 && lane == 0) {
    // ------------------------------------------------------------ producer
    int issued = 0;
    bool ok = true;
    const int end = g.starve ? kb0 : kb1;
    for (int kb = kb0; kb < end; ++kb) {
      const int i = kb - kb0, s = i % STAGES;
      if (i >= STAGES) {
        ok = mbar_wait(smem_u32(&ctrl->empty[s]), uint32_t(i / STAGES - 1) & 1u, abort_flag);
        if (!ok) break;
      }
      const uint32_t bar = smem_u32(&ctrl->full[s]), dst = smem_base + uint32_t(s * STAGE_BYTES);
      mbar_arrive_expect_tx(bar, STAGE_BYTES);
      Tiles::load_a(dst, &map_a, bar, kb, f0, 0);
      if constexpr (B_MN && BN == 64) tma_load_3d(dst + TILE_BYTES, &map_b, bar, c0, kb * Tiles::BKE, 0);
      else Tiles::load_b(dst + TILE_BYTES, &map_b, bar, kb, c0, 0);
      issued = i + 1;
    }
    if (!ok) {
      atomicCAS(g.status, 0u, unsigned(ST_PRODUCER_TIMEOUT) | unsigned(blockIdx.x & 0xff));
      // let the copies that were issued land before shared memory is used for anything else
      for (int i = issued > STAGES ? issued - STAGES : 0; i < issued; ++i)
        for (int spin = 0; spin < (1 << 20) && !mbar_try_wait(smem_u32(&ctrl->full[i % STAGES]), uint32_t(i / STAGES) & 1u); ++spin) {
        }
    }
  } else if (warp == 1 && lane == 0) {
    // ---------------------------------------------------------- MMA issuer
    bool ok = true;
    for (int kb = kb0; kb < kb1; ++kb) {
      const int i = kb - kb0, s = i % STAGES;
      ok = mbar_wait(smem_u32(&ctrl->full[s]), uint32_t(i / STAGES) & 1u, abort_flag);
      if (!ok) break;
      tc_fence_after();
      const uint32_t sa = smem_base + uint32_t(s * STAGE_BYTES);
      const uint64_t adesc = Tiles::desc_a(sa), bdesc = Tiles::desc_b(sa + TILE_BYTES);
#pragma unroll
      for (int ks = 0; ks < 4; ++ks)
        umma<KIND_F16>(tmem_base, adesc + uint64_t(ks) * Tiles::A_STEP, bdesc + uint64_t(ks) * Tiles::B_STEP, IDESC, i > 0 || ks > 0);
      umma_commit(smem_u32(&ctrl->empty[s]));
    }
    if (ok) umma_commit(smem_u32(&ctrl->acc_full[0]));
    else atomicCAS(g.status, 0u, unsigned(ST_MMA_TIMEOUT) | unsigned(blockIdx.x & 0xff));
  } else if (warp >= 4) {
    // ------------------------------------------------- accumulator to shared memory
    const bool ok = mbar_wait_warp(smem_u32(&ctrl->acc_full[0]), 0u, abort_flag);
    if (ok) {
      // The accumulator is complete: every copy of this CTA has landed and been read, the ring is free.
      tc_fence_after();
      const int q = warp & 3;
      const uint32_t own = smem_base + uint32_t(q * 32 + lane) * 4u;
#pragma unroll 1
      for (int c = 0; c < TMEM_COLS; c += 32) {
        uint32_t v[32];
        tmem_ld32(tmem_base + (uint32_t(q * 32) << 16) + uint32_t(c), v);
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (c + j < BN) sts32(own + uint32_t((c + j) * LSP_PARK_PITCH) * 4u, __uint_as_float(v[j]));
      }
    } else if (lane == 0) {
      atomicCAS(g.status, 0u, unsigned(ST_EPILOGUE_TIMEOUT) | unsigned(blockIdx.x & 0xff));
    }
  }
  // every thread comes here, whatever happened to its role; a CTA whose wait ran out has posted the status word, and the
  // columns it contributes to are meaningless but in bounds
  __syncwarp();
  tc_fence_before();
  cluster_sync();
  if (warp == 1) tmem_dealloc(tmem_base, TMEM_COLS);

  const int columns = min(BN, g.columns - c0), f = f0 + 4 * lane;
  for (int i = warp; rank + split * i < columns; i += LSP_THREADS / 32) {
    const int c = rank + split * i;
    const uint32_t at = smem_base + uint32_t(c * LSP_PARK_PITCH + 4 * lane) * 4u;
    float z[4] = {0.f, 0.f, 0.f, 0.f};
    float4 part[8];
#pragma unroll
    for (int s = 0; s < 8; ++s)
      if (s < split) part[s] = ldc128(cluster_map(at, uint32_t(s)));
#pragma unroll
    for (int s = 0; s < 8; ++s)
      if (s < split) { z[0] += part[s].x; z[1] += part[s].y; z[2] += part[s].z; z[3] += part[s].w; }
    linear_column<E>(args, g, c0 + c, f, z, lane);
  }
  cluster_sync();                    // nobody leaves while its partial tile is still being read
}

}  // namespace i8m

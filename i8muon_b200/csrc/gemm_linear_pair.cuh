// Whole-K products of a linear layer on pairs of SMs.
//
// A cluster of two CTAs takes units of 256 x 256 outputs with tcgen05.mma.cta_group::2: one instruction, issued by the first
// CTA, multiplies 256 rows of A - 128 in each CTA's shared memory - with 256 rows of B, of which each CTA holds half, and
// leaves 128 x 256 outputs in each CTA's tensor memory.  Against wholek_wide_kernel, whose CTA needs 48 KB of operands for the
// same 128 x 256 outputs of a K block, a CTA takes in 32 KB: two thirds of the traffic from L2 and of the writes to shared
// memory, which at the power limit is clock rate as well.  8192 x 2048 -> 8192 BF16: 206 -> 185 us in a burst, 225 -> 215 us
// over half a second (a library product: 176 and 205); with an INT8 copy of the pre-activation 247 -> 203 in a burst.
// What bounds it: the tensor pipe, 85 % of the active cycles (a K block takes 595 cycles for 512 of tensor work; a library product
// of these sizes 85.5 %).  An epilogue with GELU costs 14 % (74 %), an INT8 copy of the pre-activation 8 % (79 %): they run
// beside the K loop of the next unit, the last one of a CTA alone.
//
//   warp 0         TMA producer of each CTA: its 128 rows of A and its 128 rows of B, six 32 KB stages.  All copies of both CTAs
//                  count on the first CTA's barrier (their completion is what the issuer waits for)
//   warp 1         of the first CTA: tcgen05.mma issuer; its commits free a stage, and hand over an accumulator, in both CTAs
//   warps 4..19    epilogue of each CTA over its own two tiles, 32 rows x 64 columns of a unit each; both CTAs' warps free an
//                  accumulator on the first CTA's barrier.  Sixteen warps instead of eight, because a warp's chain from tensor
//                  memory to the store issues an instruction every eight to ten cycles: with K = 64, 16384 x 8192 outputs took
//                  93 us with eight, 73 with sixteen, 56 with the epilogue as it stands (a library product: 48)
// Two accumulators of 256 columns ping-pong.  Every wait is bounded, as in the other kernels; both CTAs meet before they leave.
#pragma once
#include "epi_linear.cuh"
#include "gemm_fp32_cluster.cuh"
#include "gemm_wholek_wide.cuh"

namespace i8m {

constexpr int LPR_STAGES = 6;
constexpr int LPR_STAGE_BYTES = 2 * TILE_BYTES;
constexpr int LPR_EPI_WARPS = 16;
constexpr int LPR_THREADS = 32 * (4 + LPR_EPI_WARPS);
// 640 threads are launched with 96 registers each (65536 / 640, in eights): 61440, of which these take 60416.  The host checks what
// the kernel was compiled to before its first launch: with fewer, the wait for registers would not end.
constexpr int LPR_CTRL_REGS = 56, LPR_EPI_REGS = 104;
constexpr int LPR_REGS = 32 * (4 * LPR_CTRL_REGS + LPR_EPI_WARPS * LPR_EPI_REGS);
static_assert(LPR_REGS <= LPR_THREADS * (65536 / LPR_THREADS / 8 * 8), "registers");
constexpr size_t LPR_SMEM = size_t(LPR_STAGES) * LPR_STAGE_BYTES + sizeof(Ctrl) + LPR_EPI_WARPS * WARP_PATCH_BYTES + 1024;
static_assert(LPR_SMEM <= 227 * 1024, "shared memory of a CTA");

// Unit `linear` of the pairs of row tiles x pairs of column tiles, in the grouped order of decode_unit.
__host__ __device__ __forceinline__ void decode_pair(const GemmGeom& g, int linear, int& row_pair, int& col_pair) {
  const unsigned row_pairs = unsigned(g.tiles_m + 1) / 2, cols = unsigned(g.tiles_n + 1) / 2, group = unsigned(g.group) / 2;
  const unsigned per_group = group * cols, grp = unsigned(linear) / per_group, in_group = unsigned(linear) - grp * per_group;
  const unsigned rows = row_pairs - grp * group < group ? row_pairs - grp * group : group;
  col_pair = int(in_group / rows);
  row_pair = int(grp * group + in_group % rows);
}

// Item `linear` of the units x parts of the sum: its unit and its run of K blocks.  Without PARTS a sum is whole.
struct PairItem { int row_pair, col_pair, part, kb0, kb1; };
template <bool PARTS>
__host__ __device__ __forceinline__ PairItem decode_item(const GemmGeom& g, int part_count, int linear) {
  PairItem it{0, 0, 0, 0, g.num_kb};
  if (PARTS) {
    const int unit = linear / part_count;
    it.part = linear - unit * part_count;
    it.kb0 = int((long long)g.num_kb * it.part / part_count);
    it.kb1 = int((long long)g.num_kb * (it.part + 1) / part_count);
    linear = unit;
  }
  decode_pair(g, linear, it.row_pair, it.col_pair);
  return it;
}

__device__ __forceinline__ void pair_tmem_alloc(uint32_t dst_smem, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst_smem), "r"(ncols) : "memory");
}
__device__ __forceinline__ void pair_tmem_relinquish() { asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void pair_tmem_dealloc(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
// A tiled load into this CTA's shared memory whose bytes count on a barrier of either CTA of the pair.
__device__ __forceinline__ void pair_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2"
      " [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(0)
      : "memory");
}
template <typename E, int MN>
__device__ __forceinline__ void pair_load_tile(uint32_t dst, const CUtensorMap* map, uint32_t bar, int kb, int r0) {
  using Tiles = OperandTiles<E, MN, MN>;
  if constexpr (!MN) {
    pair_load_3d(dst, map, bar, kb * Tiles::BKE, r0);
  } else {
    pair_load_3d(dst, map, bar, r0, kb * Tiles::BKE);
    pair_load_3d(dst + Tiles::MN_BOX_BYTES, map, bar, r0 + 64, kb * Tiles::BKE);
  }
}
__device__ __forceinline__ void pair_umma(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Arrive on the barrier at this offset in both CTAs once everything issued so far has been done.
__device__ __forceinline__ void pair_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
               "h"(uint16_t(3)) : "memory");
}
// Arrive on a barrier of either CTA.  What it hands over is tensor memory that has been read (ordered by tcgen05's own fence), so
// the release is left at CTA scope: at cluster scope the warp would wait here until its stores to global memory have arrived.
__device__ __forceinline__ void pair_arrive(uint32_t mapped_bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(mapped_bar) : "memory");
}

// A product whose units are fewer than the pairs, or fill their last wave badly, is cut along K: a pair takes one part of a unit's K
// blocks and parks FP32 sums, which parts_fold_kernel adds up in the order of the parts.  The gradient of 512 x 512 weights over
// 65536 rows is four units: 38.5 us in 18 parts of each, 58.8 with the split kernel (8 CTAs per tile of 128 x 64), whose tiles
// read the operands twice as often (a library product: 39.7).  An instantiation of its own (PARTS): as a run-time branch it
// cost products with short sums 5 to 10 %.
template <typename E>
__global__ void __launch_bounds__(256)
parts_fold_kernel(const float* __restrict__ parts, E* __restrict__ out, int part_count, int rows, int width, int pitch, bool vectors) {
  pdl_wait();
  const int octets = pitch / 8;
  const long long total = (long long)rows * octets, apart = (long long)rows * pitch;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
    const long long row = i / octets;
    const int col = int(i - row * octets) * 8;
    float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int p = 0; p < part_count; ++p) {
      const float4* f = reinterpret_cast<const float4*>(parts + p * apart + row * pitch + col);
      const float4 a = f[0], b = f[1];
      s[0] += a.x; s[1] += a.y; s[2] += a.z; s[3] += a.w;
      s[4] += b.x; s[5] += b.y; s[6] += b.z; s[7] += b.w;
    }
    E* to = out + row * width + col;
    if (vectors) {
      store8<E>(to, s);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (col + j < width) to[j] = round_to<E>(s[j]);
    }
  }
}

template <typename E, int A_MN, int B_MN, bool PARTS>
__global__ void __launch_bounds__(LPR_THREADS, 1)
linear_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                   const __grid_constant__ CUtensorMap map_y, const __grid_constant__ CUtensorMap map_z, GemmGeom g, LinearArgs args) {
  using Epi = EpiLinear<E>;
  using Tiles = OperandTiles<E, A_MN, B_MN>;
  constexpr int STAGES = LPR_STAGES, STAGE_BYTES = LPR_STAGE_BYTES, ACC_COLS = 2 * TILE;
  constexpr uint32_t IDESC = make_idesc(1u, Epi::FMT, Epi::FMT, 2 * TILE, 2 * TILE) | Tiles::IDESC_BITS;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* patches = smem + STAGES * STAGE_BYTES;            // on 512 bytes: the swizzle of what leaves
  Ctrl* ctrl = reinterpret_cast<Ctrl*>(patches + LPR_EPI_WARPS * WARP_PATCH_BYTES);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = int(blockIdx.x) & 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(smem_u32(&ctrl->full[s]), 1);
      mbar_init(smem_u32(&ctrl->empty[s]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&ctrl->acc_full[i]), 1);
      mbar_init(smem_u32(&ctrl->acc_empty[i]), 2 * LPR_EPI_WARPS);   // both CTAs' epilogue warps
    }
    ctrl->abort = 0;
    fence_mbar_init();
    tma_prefetch_desc(&map_a);
    tma_prefetch_desc(&map_b);
  }
  if (warp == 1) {
    pair_tmem_alloc(smem_u32(&ctrl->tmem_base), ACC_COLS * 2);
    pair_tmem_relinquish();
  }
  tc_fence_before();
  cluster_sync();                    // the barriers of both CTAs exist
  tc_fence_after();
  pdl_wait();
  const uint32_t tmem_base = ctrl->tmem_base, smem_base = smem_u32(smem);
  volatile uint32_t* abort_flag = &ctrl->abort;
  const uint32_t full0 = smem_u32(&ctrl->full[0]), empty0 = smem_u32(&ctrl->empty[0]);
  const uint32_t accf0 = smem_u32(&ctrl->acc_full[0]), acce0 = smem_u32(&ctrl->acc_empty[0]);

  const int units = (g.tiles_m + 1) / 2 * ((g.tiles_n + 1) / 2) * (PARTS ? args.part_count : 1), pairs = int(gridDim.x) / 2, pair_of = int(blockIdx.x) / 2;
  const int my_units = (units - pair_of + pairs - 1) / pairs;

  if (warp < 4) {
    setmaxnreg_dec<LPR_CTRL_REGS>();
    if (warp == 0 && lane == 0) {
      // ------------------------------------------------------------ producer
      const uint32_t full_at = cluster_map(full0, 0);        // the first CTA's barriers
      int ring = 0, issued = 0;
      uint32_t wrap = 0;
      bool ok = true;
      const int todo = (g.debug_simt & 0x100) ? 0 : my_units;  // test hook: issue nothing
      for (int j = 0; j < todo && ok; ++j) {
        const PairItem it = decode_item<PARTS>(g, args.part_count, pair_of + j * pairs);
        const int r0 = (2 * it.row_pair + rank) * TILE, n0 = (2 * it.col_pair + rank) * TILE;
        for (int kb = it.kb0; kb < it.kb1; ++kb) {
          if (wrap > 0) {
            ok = mbar_wait(empty0 + 8u * uint32_t(ring), (wrap - 1) & 1u, abort_flag);
            if (!ok) break;
          }
          const uint32_t dst = smem_base + uint32_t(ring * STAGE_BYTES), bar = full_at + 8u * uint32_t(ring);
          if (rank == 0) mbar_arrive_expect_tx(full0 + 8u * uint32_t(ring), 2 * STAGE_BYTES);
          pair_load_tile<E, A_MN>(dst, &map_a, bar, kb, r0);
          pair_load_tile<E, B_MN>(dst + TILE_BYTES, &map_b, bar, kb, n0);
          ++issued;
          if (++ring == STAGES) { ring = 0; ++wrap; }
        }
      }
      if (!ok) {
        atomicCAS(g.status, 0u, unsigned(ST_PRODUCER_TIMEOUT) | unsigned(blockIdx.x & 0xff));
        // let what was issued land (it counts on the first CTA's barriers, which only that CTA can watch)
        for (int back = 0; rank == 0 && back < STAGES && back < issued; ++back) {
          const int n = issued - 1 - back;
          for (int spin = 0; spin < (1 << 20) && !mbar_try_wait(full0 + 8u * uint32_t(n % STAGES), uint32_t(n / STAGES) & 1u); ++spin) {
          }
        }
      }
    } else if (warp == 1 && lane == 0 && rank == 0) {
      // ---------------------------------------------------------- MMA issuer of the pair
      int ring = 0;
      uint32_t wrap = 0;
      bool ok = true;
      for (int j = 0; j < my_units && ok; ++j) {
        const int buf = j & 1;
        const uint32_t use = uint32_t(j >> 1);
        if (use >= 1) {
          ok = mbar_wait(acce0 + 8u * uint32_t(buf), (use - 1) & 1u, abort_flag);
          if (!ok) break;
          tc_fence_after();
        }
        const uint32_t d = tmem_base + uint32_t(buf * ACC_COLS);
        const PairItem it = decode_item<PARTS>(g, args.part_count, pair_of + j * pairs);
        for (int kb = it.kb0; kb < it.kb1; ++kb) {
          ok = mbar_wait(full0 + 8u * uint32_t(ring), wrap & 1u, abort_flag);
          if (!ok) break;
          tc_fence_after();
          const uint32_t sa = smem_base + uint32_t(ring * STAGE_BYTES);
          const uint64_t adesc = Tiles::desc_a(sa), bdesc = Tiles::desc_b(sa + TILE_BYTES);
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
            pair_umma(d, adesc + uint64_t(ks) * Tiles::A_STEP, bdesc + uint64_t(ks) * Tiles::B_STEP, IDESC, kb > it.kb0 || ks > 0);
          pair_commit(empty0 + 8u * uint32_t(ring));
          if (++ring == STAGES) { ring = 0; ++wrap; }
        }
        if (ok) pair_commit(accf0 + 8u * uint32_t(buf));
      }
      if (!ok) atomicCAS(g.status, 0u, unsigned(ST_MMA_TIMEOUT) | unsigned(blockIdx.x & 0xff));
    }
  } else {
    // -------------------------------------------------------------- epilogue
    setmaxnreg_inc<LPR_EPI_REGS>();
    const uint32_t freed = cluster_map(acce0, 0);            // the first CTA's barriers
    TileCtx t;
    t.b = 0;
    t.q = warp & 3; t.lane = lane;
    t.ew = warp - 4;
    const int slice = t.ew >> 2;                             // of the unit's 256 columns: 64
    t.half = slice & 1;
    t.r = t.q * 32 + lane;
    t.ctrl = ctrl;
    t.red = ctrl->red; t.diag = ctrl->diag;
    t.tsm = nullptr;
    t.wsm = patches + t.ew * WARP_PATCH_BYTES;
    t.c_begin = t.half * 2; t.c_end = t.half * 2 + 2;
    bool ok = true;
    PairItem next{};
    auto decode_next = [&](int j) {
      next = decode_item<PARTS>(g, args.part_count, pair_of + j * pairs);
      Epi::expect_residual(g, args, (2 * next.row_pair + rank) * TILE + t.r, 2 * next.col_pair * TILE + 64 * slice);
    };
    if (my_units > 0) decode_next(0);
    for (int j = 0; j < my_units; ++j) {
      const PairItem it = next;
      if (j + 1 < my_units) decode_next(j + 1);
      t.tm = 2 * it.row_pair + rank;
      t.row0 = t.tm * TILE;
      t.row = t.row0 + t.r;
      const int buf = j & 1;
      ok = mbar_wait_warp(accf0 + 8u * uint32_t(buf), uint32_t(j >> 1) & 1u, abort_flag);
      if (!ok) break;
      tc_fence_after();
      t.tn = 2 * it.col_pair + (slice >> 1);
      t.col0 = t.tn * TILE;
      AccWholeK<KIND_F16, E, false> acc{g, t, tmem_base + (uint32_t(t.q * 32) << 16) + uint32_t(buf * ACC_COLS + (slice >> 1) * TILE)};
      if constexpr (PARTS) Epi::park(g, args, it.part, t, acc);
      else Epi::run(g, args, &map_y, &map_z, t, acc);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) pair_arrive(freed + 8u * uint32_t(buf));
    }
    Epi::patch_free(WarpPatch{smem_u32(t.wsm), lane});       // copies from it end before the CTA does
    if (!ok && lane == 0) atomicCAS(g.status, 0u, unsigned(ST_EPILOGUE_TIMEOUT) | unsigned(blockIdx.x & 0xff));
  }
  __syncwarp();
  tc_fence_before();
  cluster_sync();                    // neither CTA leaves while the other may signal its barriers or multiply its operands
  if (warp == 1) pair_tmem_dealloc(tmem_base, ACC_COLS * 2);
}

}  // namespace i8m

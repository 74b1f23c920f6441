// C ABI: linear layers (product with bias, activation and residual in the epilogue) and their backward pass.
#include "launch_gemm.cuh"
#include "epi_linear.cuh"
#include "gemm_linear_pair.cuh"
#include "gemm_linear_split.cuh"
#include "layers.cuh"

#include <algorithm>
#include <cmath>

using namespace i8m;

namespace {

// An operand: `extent` rows along K, or (mn) K rows along its extent; rows `pitch` elements apart.
struct Operand {
  const void* p;
  int pitch, mn;
};

// How a product is carried out: on pairs of SMs in units of 256 x 256 (bn 0), K cut into `split` parts, or by the split kernel with
// tiles of 128 features x bn rows and K cut over `split` CTAs.
struct Plan {
  int bn, split;
};
// Parts are FP32 results in the workspace, at most this much.
constexpr size_t MOST_PART_BYTES = size_t(64) << 20;
inline size_t part_bytes(int m, int n) { return size_t(m) * pad_to(n, 8) * 4; }
// The least of an estimate in nanoseconds.  Pairs: 6 us, and 0.365 us per K block of a wave of units, at least 1.85 us (an epilogue)
// for every wave but the first; in parts, 3 us more for the launch that folds them and 8 TB/s for what it moves.  Split kernel: 4.5 us and 25 ns
// per column of the tile for its start, sums and end, 4 us for every further wave, and per K block 14 ns for each KB that the
// CTA takes in, at least 0.27 us, or 17 ns per KB where two CTAs share an SM.  Both: beside the time that DRAM takes for the
// operands (as the root of the sum of squares: neither hides the other fully).
// Measured with BF16 operands beyond L2, in us, pairs / best split (bn, CTAs per tile): 1 x 4096 -> 4096 25 / 10.4 (16, 4);
// 16 x 4096 -> 14336 29 / 23.6 (16, 2); 256 x 4096 -> 4096 26.6 / 17.2 (128, 4); 512 27.2 / 23.1 (128, 2); 1024 28.7 / 37.6 (128, 1);
// 333 x 1008 -> 520 11.4 / 6.5 (64, 4); 1024 x 768 -> 768 10.2 / 9.0 (32, 1); 2048 x 1024 -> 1024 12.3 / 12.9 (64, 1);
// 300 x 8192 -> 256 44.6 / 10.8 (64, 8).
Plan plan_product(int rows, int features, int k, bool rows_mn, int sms, size_t room) {
  const int num_kb = cdiv(2LL * k, 128);
  const double dram = 2.0 * k * ((double)rows + features) / 6200.0;
  auto beside_dram = [&](double v) { return std::sqrt(v * v + dram * dram); };
  const long long units = (long long)cdiv(rows, 2 * TILE) * cdiv(features, 2 * TILE), pairs = std::max(1, sms / 2);
  Plan best{0, 1};
  double cost = 1e30;
  for (int parts = 1; parts <= 64 && (parts == 1 || (4 * parts <= num_kb && parts * part_bytes(rows, features) <= room)); ++parts) {
    const double block = (num_kb + parts - 1) / parts * 365.0, fold = 3000 + 2.0 * parts * part_bytes(rows, features) / 8000.0;
    const double c = 6000 + beside_dram(block + ((units * parts + pairs - 1) / pairs - 1) * std::max(1850.0, block)) + (parts > 1 ? fold : 0);
    if (c < cost) { cost = c; best = {0, parts}; }
  }
  for (int bn = rows_mn ? 64 : 16; bn <= 128; bn *= 2) {
    const long long split_tiles = (long long)cdiv(features, TILE) * cdiv(rows, bn), kilobytes = 16 + bn / 8;
    for (int split = 1; split <= 8 && split <= num_kb; split *= 2) {
      // CTAs resident at one time, two per SM: GPC sizes leave some SMs out of larger clusters (148, 74, 33, 15 clusters measured)
      const int resident = sms * 2 * (split == 4 ? 132 : split == 8 ? 120 : 148) / 148;
      const long long ctas = split_tiles * split, waves = (ctas + resident - 1) / resident;
      if (waves > 4) break;
      const long long block = ctas > sms ? 17 * kilobytes : std::max<long long>(270, 14 * kilobytes);
      const double c = 4500 + 25 * bn + 4000.0 * (waves - 1) + beside_dram(double(waves * ((num_kb + split - 1) / split) * block));
      if (c < cost) { cost = c; best = {bn, split}; }
    }
    if (bn >= rows) break;
  }
  return best;
}

template <typename E, int BN, int A_MN, int B_MN>
int launch_split(const CUtensorMap& ma, const CUtensorMap& mb, const LinearSplitGeom& g, const LinearArgs& args, cudaStream_t stream,
                 const char* name) {
  auto kernel = linear_split_kernel<E, BN, A_MN, B_MN>;
  constexpr size_t SMEM = LinearSplitShape<BN>::SMEM;
  static SmemAllowed allowed;
  if (int rc = allow_smem(allowed, kernel, SMEM)) return rc;
  const unsigned grid = unsigned(g.tiles_f * cdiv(g.columns, BN) * g.split);
  launch_clusters(kernel, unsigned(g.split), grid, LSP_THREADS, SMEM, stream, ma, mb, g, args);
  LAUNCH_CHECK(name);
  return 0;
}
template <typename E, int BN>
int launch_split_layout(int f_mn, int c_mn, const CUtensorMap& ma, const CUtensorMap& mb, const LinearSplitGeom& g,
                        const LinearArgs& args, cudaStream_t stream, const char* name) {
  if (!f_mn) return launch_split<E, BN, 0, 0>(ma, mb, g, args, stream, name);
  if constexpr (BN >= 64) {
    if (c_mn) return launch_split<E, BN, 1, 1>(ma, mb, g, args, stream, name);
  }
  return launch_split<E, BN, 1, 0>(ma, mb, g, args, stream, name);
}
// out (m, n) with the split kernel: n are the features, b their operand.
template <typename E>
int product_split(const Plan& plan, const Operand& a, const Operand& b, int m, int n, int k, const LinearArgs& args, unsigned* status,
                  cudaStream_t stream, const char* name) {
  LinearSplitGeom g{n, m, cdiv(2LL * k, 128), cdiv(n, TILE), plan.split, g_starve_producers, status};
  CUtensorMap mf, mc;
  if (int rc = make_operand_map(&mf, b.p, 2, k, n, 1, b.mn, b.pitch)) return rc;
  if (int rc = make_operand_map(&mc, a.p, 2, k, m, 1, a.mn, a.pitch, plan.bn)) return rc;
  switch (plan.bn) {
    case 16: return launch_split_layout<E, 16>(b.mn, a.mn, mf, mc, g, args, stream, name);
    case 32: return launch_split_layout<E, 32>(b.mn, a.mn, mf, mc, g, args, stream, name);
    case 64: return launch_split_layout<E, 64>(b.mn, a.mn, mf, mc, g, args, stream, name);
    default: return launch_split_layout<E, 128>(b.mn, a.mn, mf, mc, g, args, stream, name);
  }
}

// Rows of `width` 16-bit elements, one behind the other, that tensor copies can address.
bool addressable(const void* p, int width) { return width % 8 == 0 && (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <typename E, int A_MN, int B_MN, bool PARTS = false>
int launch_pair(const CUtensorMap& ma, const CUtensorMap& mb, const GemmGeom& g, LinearArgs args, unsigned pairs,
                cudaStream_t stream, const char* name) {
  CUtensorMap my = ma, mz = ma;          // what is not stored through its map has none
  args.y_blocks = !PARTS && addressable(args.y, g.n);
  if (args.y_blocks)
    if (int rc = make_block_map(&my, args.y, g.n, g.m, g.n)) return rc;
  if (args.z != nullptr)
    if (int rc = make_block_map(&mz, args.z, args.z_pitch, g.m, args.z_pitch)) return rc;
  auto kernel = linear_pair_kernel<E, A_MN, B_MN, PARTS>;
  static SmemAllowed allowed;
  if (int rc = allow_smem(allowed, kernel, LPR_SMEM)) return rc;
  static const int registers = [&] {
    cudaFuncAttributes attributes;
    return cudaFuncGetAttributes(&attributes, kernel) == cudaSuccess ? attributes.numRegs : 0;
  }();
  if (registers * LPR_THREADS < LPR_REGS) return fail(I8M_E_CUDA, "%s: compiled to %d registers, too few to share out", name, registers);
  launch_clusters(kernel, 2, 2 * pairs, LPR_THREADS, LPR_SMEM, stream, ma, mb, my, mz, g, args);
  LAUNCH_CHECK(name);
  return 0;
}

// out (m, n) = a b^T over k.  `parts`: room for FP32 parts of it, of `room` bytes (none: the sum stays whole).
template <typename E>
int product(const Operand& a, const Operand& b, int m, int n, int k, LinearArgs args, float* parts, size_t room, unsigned* status,
            cudaStream_t stream, const char* name) {
  GemmGeom g{};
  g.batch = 1; g.m = g.lm = m; g.n = g.ln = n; g.k = k;
  g.tiles_m = cdiv(m, TILE); g.tiles_n = cdiv(n, TILE);
  const long long tiles = (long long)g.tiles_m * g.tiles_n;
  if (tiles > 0x7fffffffLL) return fail(I8M_E_LIMIT, "%s: too many tiles", name);
  g.tiles_per_batch = int(tiles);
  g.num_kb = cdiv(2LL * k, 128);
  g.debug_simt = g_starve_producers ? 0x100 : 0;
  g.a_mn = a.mn; g.b_mn = b.mn;
  g.group = wide_group(2LL * k);
  g.a_raw = a.p; g.b_raw = b.p; g.status = status;
  const Plan plan = plan_product(m, n, k, a.mn, sm_count(), room);
  if (plan.bn) return product_split<E>(plan, a, b, m, n, k, args, status, stream, name);
  CUtensorMap ma, mb;
  if (int rc = make_operand_map(&ma, a.p, 2, k, m, 1, a.mn, a.pitch)) return rc;
  if (int rc = make_operand_map(&mb, b.p, 2, k, n, 1, b.mn, b.pitch)) return rc;
  const long long units = (long long)cdiv(g.tiles_m, 2) * cdiv(g.tiles_n, 2);
  const unsigned pairs_of_sms = unsigned(std::min<long long>(units * plan.split, std::max(1, sm_count() / 2)));
  if (plan.split == 1) {
    if (!a.mn && !b.mn) return launch_pair<E, 0, 0>(ma, mb, g, args, pairs_of_sms, stream, name);
    if (!a.mn) return launch_pair<E, 0, 1>(ma, mb, g, args, pairs_of_sms, stream, name);
    return launch_pair<E, 1, 1>(ma, mb, g, args, pairs_of_sms, stream, name);
  }
  args.parts = parts; args.part_count = plan.split; args.z_pitch = pad_to(n, 8);
  if (int rc = a.mn ? launch_pair<E, 1, 1, true>(ma, mb, g, args, pairs_of_sms, stream, name)      // room is given to gradients alone
                    : launch_pair<E, 0, 1, true>(ma, mb, g, args, pairs_of_sms, stream, name)) return rc;
  const long long octets = (long long)m * (args.z_pitch / 8);
  launch(parts_fold_kernel<E>, unsigned(std::min<long long>((octets + 255) / 256, 148LL * 8)), 256, 0, stream, parts, static_cast<E*>(args.y),
         plan.split, m, n, args.z_pitch, addressable(args.y, n));
  LAUNCH_CHECK("parts_fold");
  return 0;
}
template <typename... A>
int product_of(int dtype, A&&... args) {
  return dtype == I8M_F16 ? product<__half>(std::forward<A>(args)...) : product<__nv_bfloat16>(std::forward<A>(args)...);
}

// Extents come as 64-bit numbers: what a caller passes is what is compared with the limits.
int check_linear(const char* name, long long rows, long long inner, long long outer, int dtype, int activation, int format) {
  if (rows < 1 || inner < 1 || outer < 1) return fail(I8M_E_ARGUMENT, "%s: empty problem", name);
  if (dtype != I8M_F16 && dtype != I8M_BF16) return fail(I8M_E_ARGUMENT, "%s: dtype must be a 16-bit type", name);
  if (activation < 0 || activation >= ACTIVATIONS) return fail(I8M_E_ARGUMENT, "%s: bad activation %d", name, activation);
  if (format < -1 || format > EIGHT_E4M3) return fail(I8M_E_ARGUMENT, "%s: bad format %d", name, format);
  if (inner > MAX_LAYER_WIDTH || outer > MAX_LAYER_WIDTH || rows > MAX_LAYER_ROWS)
    return fail(I8M_E_LIMIT, "%s: %lld rows, %lld x %lld weights are above the limits", name, rows, outer, inner);
  return 0;
}

// Workspace: pieces one behind the other, each aligned to 256 bytes.
struct Carver {
  uint8_t* base;
  size_t used = 0;
  void* take(size_t bytes) {
    void* p = base + used;
    used += align256(bytes);
    return p;
  }
};
size_t rows_bytes(long long rows, int pitch) { return size_t(rows) * pitch * 2; }

// What a forward or backward call copies or computes into its workspace.
struct ForwardPieces {
  void *x = nullptr, *w = nullptr;
  size_t bytes;
  ForwardPieces(void* base, const void* x_in, const void* w_in, int rows, int inner, int outer) {
    Carver c{static_cast<uint8_t*>(base)};
    const int pitch = pad_to(inner, 8);
    if (!addressable(x_in, inner)) x = c.take(rows_bytes(rows, pitch));
    if (!addressable(w_in, inner)) w = c.take(rows_bytes(outer, pitch));
    bytes = c.used;
  }
};
struct BackwardPieces {
  void *w = nullptr, *x = nullptr, *dz = nullptr;
  float *partials = nullptr, *parts = nullptr;
  size_t bytes, room = 0;
  BackwardPieces(void* base, const void* dy, const void* x_in, const void* w_in, int rows, int inner, int outer, int activation,
                 int format, bool dx, bool dw, bool db) {
    Carver c{static_cast<uint8_t*>(base)};
    const int pitch = pad_to(inner, 8);
    if (dx && !addressable(w_in, inner)) w = c.take(rows_bytes(outer, pitch));
    if (dw && (format >= 0 || !addressable(x_in, inner))) x = c.take(rows_bytes(rows, pitch));
    if ((dx || dw) && (activation != ACT_NONE || !addressable(dy, outer))) dz = c.take(rows_bytes(rows, pad_to(outer, 8)));
    if (db) partials = static_cast<float*>(c.take(size_t(dz_bands(rows, outer)) * 2 * outer * sizeof(float)));
    // a product may be cut for 148 SMs; where fewer are in use it is cut to fit
    auto parts_of = [&](int m, int n, int k, bool mn) {
      const Plan plan = plan_product(m, n, k, mn, 148, MOST_PART_BYTES);
      return plan.bn == 0 && plan.split > 1 ? plan.split * part_bytes(m, n) : size_t(0);
    };
    if (dx) room = parts_of(rows, inner, outer, false);
    if (dw) room = std::max(room, parts_of(outer, inner, rows, true));
    if (room) parts = static_cast<float*>(c.take(room));
    bytes = c.used;
  }
};

}  // namespace

extern "C" int i8m_linear_workspace_bytes(const void* x, const void* weight, long long rows, long long inner, long long outer,
                                          size_t* bytes) {
  if (!bytes) return fail(I8M_E_ARGUMENT, "linear_workspace_bytes: null pointer");
  if (int rc = check_linear("linear_workspace_bytes", rows, inner, outer, I8M_BF16, 0, -1)) return rc;
  *bytes = ForwardPieces(nullptr, x, weight, int(rows), int(inner), int(outer)).bytes;
  return 0;
}
extern "C" int i8m_linear(const void* x, const void* weight, const void* bias, const void* residual, void* y, void* z,
                          void* z_codes, void* z_exponents, int format, int activation, long long row_count, long long inner_width,
                          long long outer_width, int dtype, void* workspace, size_t workspace_bytes, uint32_t* status,
                          i8m_stream_t stream) {
  if (!x || !weight || !y || !status) return fail(I8M_E_ARGUMENT, "linear: null pointer");
  if (int rc = check_linear("linear", row_count, inner_width, outer_width, dtype, activation, format)) return rc;
  const int rows = int(row_count), inner = int(inner_width), outer = int(outer_width);
  if (format >= 0 && !z_codes != !z_exponents) return fail(I8M_E_ARGUMENT, "linear: codes without exponents");
  if ((reinterpret_cast<uintptr_t>(z) | (format >= 0 ? reinterpret_cast<uintptr_t>(z_codes) : 0)) & 15u)
    return fail(I8M_E_ARGUMENT, "linear: z or its codes are not 16-byte aligned");
  const ForwardPieces pieces(workspace, x, weight, rows, inner, outer);
  if (pieces.bytes && (!workspace || workspace_bytes < pieces.bytes))
    return fail(I8M_E_WORKSPACE, "linear: workspace %zu < %zu bytes", workspace ? workspace_bytes : 0, pieces.bytes);
  if (pieces.bytes && (reinterpret_cast<uintptr_t>(workspace) & 15u)) return fail(I8M_E_ARGUMENT, "linear: workspace is not 16-byte aligned");
  const int pitch = pad_to(inner, 8);
  if (int rc = pitch_rows(x, pieces.x, rows, weight, pieces.w, outer, dtype, inner, pitch, S(stream))) return rc;
  LinearArgs a{};
  a.y = y; a.bias = bias; a.residual = residual;
  a.z = format < 0 ? z : nullptr; a.z_pitch = pad_to(outer, 8);
  a.codes = format >= 0 ? static_cast<uint8_t*>(z_codes) : nullptr; a.exponents = static_cast<uint8_t*>(z_exponents);
  a.groups = eight_groups(outer); a.format = format; a.activation = activation;
  return product_of(dtype, Operand{pieces.x ? pieces.x : x, pitch, 0}, Operand{pieces.w ? pieces.w : weight, pitch, 0}, rows, outer,
                    inner, a, nullptr, size_t(0), status, S(stream), "linear");
}

extern "C" int i8m_linear_backward_workspace_bytes(const void* dy, const void* x, const void* weight, long long rows, long long inner,
                                                   long long outer, int activation, int format, int dx, int dweight, int dbias,
                                                   size_t* bytes) {
  if (!bytes) return fail(I8M_E_ARGUMENT, "linear_backward_workspace_bytes: null pointer");
  if (int rc = check_linear("linear_backward_workspace_bytes", rows, inner, outer, I8M_BF16, activation, format)) return rc;
  *bytes = BackwardPieces(nullptr, dy, x, weight, int(rows), int(inner), int(outer), activation, format, dx, dweight, dbias).bytes;
  return 0;
}
extern "C" int i8m_linear_backward(const void* dy, const void* x, const void* x_codes, const void* x_exponents, const void* weight,
                                   const void* z, const void* z_codes, const void* z_exponents, int format, int activation,
                                   void* dx, void* dweight, void* dbias, long long row_count, long long inner_width,
                                   long long outer_width, int dtype, void* workspace, size_t workspace_bytes, uint32_t* status,
                                   i8m_stream_t stream) {
  if (!dy || !status || (!dx && !dweight && !dbias)) return fail(I8M_E_ARGUMENT, "linear_backward: null pointer");
  if (int rc = check_linear("linear_backward", row_count, inner_width, outer_width, dtype, activation, format)) return rc;
  const int rows = int(row_count), inner = int(inner_width), outer = int(outer_width);
  if (dx && !weight) return fail(I8M_E_ARGUMENT, "linear_backward: dx needs the weight");
  if (dweight && (format < 0 ? !x : !x_codes || !x_exponents))
    return fail(I8M_E_ARGUMENT, "linear_backward: the weight's gradient needs x or its codes");
  if (dweight && format >= 0 && (reinterpret_cast<uintptr_t>(x_codes) & 15u))
    return fail(I8M_E_ARGUMENT, "linear_backward: codes of x are not 16-byte aligned");
  if (activation != ACT_NONE && (format < 0 ? !z : !z_codes || !z_exponents))
    return fail(I8M_E_ARGUMENT, "linear_backward: an activation needs z or its codes");
  if ((reinterpret_cast<uintptr_t>(z) | (format >= 0 ? reinterpret_cast<uintptr_t>(z_codes) : 0)) & 15u)
    return fail(I8M_E_ARGUMENT, "linear_backward: z or its codes are not 16-byte aligned");
  const BackwardPieces pieces(workspace, dy, x, weight, rows, inner, outer, activation, format, dx, dweight, dbias);
  if (pieces.bytes && (!workspace || workspace_bytes < pieces.bytes))
    return fail(I8M_E_WORKSPACE, "linear_backward: workspace %zu < %zu bytes", workspace ? workspace_bytes : 0, pieces.bytes);
  if (pieces.bytes && (reinterpret_cast<uintptr_t>(workspace) & 31u)) return fail(I8M_E_ARGUMENT, "linear_backward: workspace is not 32-byte aligned");
  const int inner_pitch = pad_to(inner, 8), outer_pitch = pad_to(outer, 8);

  if (pieces.dz || dbias) {
    LinearDz d{};
    d.dy = dy; d.z = z; d.codes = z_codes; d.exponents = z_exponents;
    d.format = format; d.activation = activation; d.dtype = dtype; d.rows = rows; d.width = outer; d.z_pitch = outer_pitch;
    d.dz = pieces.dz; d.dz_pitch = outer_pitch; d.db = dbias; d.partials = pieces.partials;
    if (int rc = linear_dz(d, S(stream))) return rc;
  }
  const bool restored = format >= 0 && dweight;      // x comes from its codes
  if (int rc = pitch_rows(x, restored ? nullptr : pieces.x, rows, weight, pieces.w, outer, dtype, inner, inner_pitch, S(stream)))
    return rc;
  const void* dz = pieces.dz ? pieces.dz : dy;
  LinearArgs a{};
  if (dx) {
    a.y = dx;
    if (int rc = product_of(dtype, Operand{dz, outer_pitch, 0}, Operand{pieces.w ? pieces.w : weight, inner_pitch, 1}, rows, inner,
                            outer, a, pieces.parts, pieces.room, status, S(stream), "linear_dx")) return rc;
  }
  if (dweight) {
    if (restored)
      if (int rc = eight_restore(x_codes, x_exponents, rows, inner, format, pieces.x, dtype, inner_pitch, S(stream))) return rc;
    a.y = dweight;
    if (int rc = product_of(dtype, Operand{dz, outer_pitch, 1}, Operand{pieces.x ? pieces.x : x, inner_pitch, 1}, outer, inner, rows,
                            a, pieces.parts, pieces.room, status, S(stream), "linear_dweight")) return rc;
  }
  return 0;
}

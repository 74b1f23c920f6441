// C ABI: layer norm.
#include "host.cuh"
#include "layers.cuh"
#include "layer_norm.cuh"

#include <initializer_list>

using namespace i8m;

// ================================================================== layer norm
namespace {

int check_norm(const char* name, const void* a, const void* b, long long rows, long long width, int dtype, const void* codes,
               const void* exponents, int format) {
  if (!a || !b) return fail(I8M_E_ARGUMENT, "%s: null pointer", name);
  if (rows < 1 || width < 1) return fail(I8M_E_ARGUMENT, "%s: empty problem", name);
  if (!float_dtype_ok(dtype)) return fail(I8M_E_ARGUMENT, "%s: bad dtype %d", name, dtype);
  if (format < -1 || format > EIGHT_E4M3) return fail(I8M_E_ARGUMENT, "%s: bad format %d", name, format);
  if (format >= 0 && (!codes || !exponents)) return fail(I8M_E_ARGUMENT, "%s: null codes or exponents", name);
  if (format >= 0 && (reinterpret_cast<uintptr_t>(codes) & 15u)) return fail(I8M_E_ARGUMENT, "%s: codes are not 16-byte aligned", name);
  if (width > MAX_LAYER_WIDTH) return fail(I8M_E_LIMIT, "%s: width %lld is above %d", name, width, MAX_LAYER_WIDTH);
  if (rows > MAX_LAYER_ROWS) return fail(I8M_E_LIMIT, "%s: %lld rows are above %lld", name, rows, MAX_LAYER_ROWS);
  return 0;
}
// Calls f(kernel family) for the shape.
template <bool W, int V>
struct LnFamily {
  static constexpr bool WARP = W;
  static constexpr int OCTETS = V;
};
template <int MOST, class F>
void with_ln_shape(const LnShape& s, F&& f) {
  const bool warp = s.threads == 32;
  if (warp && s.octets == 1) return f(LnFamily<true, 1>{});
  if (warp && s.octets == 2) return f(LnFamily<true, 2>{});
  if constexpr (MOST == 4) {
    if (warp && s.octets == 3) return f(LnFamily<true, 3>{});
    if (warp) return f(LnFamily<true, 4>{});
    if (s.octets == 3) return f(LnFamily<false, 3>{});
  } else {
    if (s.octets == 2) return f(LnFamily<false, 2>{});
  }
  f(LnFamily<false, 4>{});
}
// Rows that start on 16 bytes throughout.
bool ln_vectors(int width, std::initializer_list<const void*> tensors) {
  uintptr_t bits = 0;
  for (const void* p : tensors) bits |= reinterpret_cast<uintptr_t>(p);
  return width % 8 == 0 && (bits & 15u) == 0;
}
}  // namespace

extern "C" int i8m_layer_norm(const void* x, const void* weight, const void* bias, void* y, float* mean, float* rstd,
                              void* codes, void* exponents, int format, long long rows, long long row_width, int dtype, float eps,
                              i8m_stream_t stream) {
  if (int rc = check_norm("layer_norm", x, y, rows, row_width, dtype, codes, exponents, format)) return rc;
  const int width = int(row_width);
  const int groups = eight_groups(width);
  const LnShape shape = ln_shape(width, LN_FORWARD_OCTETS);
  uint8_t *c = static_cast<uint8_t*>(codes), *e = static_cast<uint8_t*>(exponents);
  if (!shape.octets) {
    const unsigned grid = unsigned(std::min<long long>(rows, 148LL * 8));
    DISPATCH_IN(dtype, E, DISPATCH_FORMAT(format, F, (launch(
        ln_forward_loop_kernel<E, F>, grid, LN_THREADS, 0, S(stream), static_cast<const E*>(x), static_cast<const E*>(weight),
        static_cast<const E*>(bias), static_cast<E*>(y), mean, rstd, c, e, rows, width, groups, eps))));
  } else {
    const bool vectors = ln_vectors(width, {x, weight, bias, format >= 0 ? codes : nullptr}) && on_octets(y, dtype_size(dtype));
    int rc = 0;
    DISPATCH_IN(dtype, E, with_ln_shape<LN_FORWARD_OCTETS>(shape, [&](auto family) {
      using Family = decltype(family);
      constexpr int V = Family::OCTETS;
      auto kernel = vectors ? ln_forward_kernel<E, Family::WARP, V, false> : ln_forward_kernel<E, Family::WARP, V, true>;
      const int block = shape.block();
      constexpr size_t STAGES = LN_STAGES<E, Family::WARP, V, 1>;
      const size_t smem = STAGES * (block * V * 8 * sizeof(E) + (vectors ? 0 : 16 * shape.rows_of_block()));
      static SmemAllowed allowed[2];
      rc = allow_smem(allowed[vectors], kernel, STAGES * (ln_stage_bytes<E, Family::WARP, V>(1) + 16 * LN_WARP_ROWS));
      if (rc) return;
      launch(kernel, unsigned(std::min<long long>(cdiv(rows, shape.rows_of_block()), 148LL * shape.resident(512, smem))), block, smem, S(stream),
             static_cast<const E*>(x), static_cast<const E*>(weight), static_cast<const E*>(bias), static_cast<E*>(y), mean, rstd,
             c, e, format, rows, width, groups, eps);
    }));
    if (rc) return rc;
  }
  LAUNCH_CHECK("layer_norm");
  return 0;
}

extern "C" int i8m_layer_norm_scratch_bytes(long long rows, long long width, size_t* bytes) {
  if (rows < 1 || width < 1 || !bytes) return fail(I8M_E_ARGUMENT, "layer_norm_scratch_bytes: bad argument");
  if (width > MAX_LAYER_WIDTH) return fail(I8M_E_LIMIT, "layer_norm_scratch_bytes: width %lld is above %d", width, MAX_LAYER_WIDTH);
  *bytes = size_t(ln_bands(rows, int(width))) * 2 * size_t(width) * sizeof(float);
  return 0;
}
extern "C" int i8m_layer_norm_backward(const void* dy, const void* x, const float* mean, const float* rstd, const void* codes,
                                       const void* exponents, int format, const void* weight, void* dx, void* dweight,
                                       void* dbias, long long rows, long long row_width, int dtype, void* scratch,
                                       size_t scratch_bytes, i8m_stream_t stream) {
  if (int rc = check_norm("layer_norm_backward", dy, rstd, rows, row_width, dtype, codes, exponents, format)) return rc;
  const int width = int(row_width);
  if (format < 0 && (!x || !mean)) return fail(I8M_E_ARGUMENT, "layer_norm_backward: neither x and its means nor codes");
  if (!dx && !dweight && !dbias) return fail(I8M_E_ARGUMENT, "layer_norm_backward: nothing to compute");
  size_t need = 0;
  if (int rc = i8m_layer_norm_scratch_bytes(rows, width, &need)) return rc;
  const bool sums = dweight || dbias;
  if (sums && (!scratch || scratch_bytes < need))
    return fail(I8M_E_WORKSPACE, "layer_norm_backward: scratch %zu < %zu bytes", scratch ? scratch_bytes : 0, need);
  const int groups = eight_groups(width);
  const LnShape shape = ln_shape(width, LN_BACKWARD_OCTETS);
  const int bands = ln_bands(rows, width);
  float* partials = static_cast<float*>(scratch);
  const uint8_t *c = static_cast<const uint8_t*>(codes), *e = static_cast<const uint8_t*>(exponents);
  if (shape.octets) {
    const bool vectors = ln_vectors(width, {dy, format < 0 ? x : codes, weight}) && on_octets(dx, dtype_size(dtype));
    int rc = 0;
    DISPATCH_IN(dtype, E, with_ln_shape<LN_BACKWARD_OCTETS>(shape, [&](auto family) {
      using Family = decltype(family);
      constexpr int V = Family::OCTETS;
      constexpr bool WARP = Family::WARP;
      const LnKept<E> kept{static_cast<const E*>(x), mean, c, e, groups};
      const E *d = static_cast<const E*>(dy), *wt = static_cast<const E*>(weight);
      float* sums_to = sums ? partials : nullptr;
      constexpr size_t STAGES = LN_STAGES<E, WARP, V, 2>, THREAD = STAGES * 2 * V * 8 * sizeof(E);
      const size_t smem = THREAD * shape.block() + (vectors ? 0 : STAGES * 2 * 16 * shape.rows_of_block());
      DISPATCH_FORMAT(format, F, {
        auto kernel = vectors ? ln_backward_kernel<E, WARP, V, F, false> : ln_backward_kernel<E, WARP, V, F, true>;
        static SmemAllowed allowed[2];
        rc = allow_smem(allowed[vectors], kernel, THREAD * (WARP ? 32 * LN_WARP_ROWS : LN_BLOCK) + STAGES * 2 * 16 * LN_WARP_ROWS);
        if (rc) return;
        launch(kernel, unsigned(bands), shape.block(), smem, S(stream), d, kept, rstd, wt, static_cast<E*>(dx), sums_to, rows, width);
      });
    }));
    if (rc) return rc;
    LAUNCH_CHECK("layer_norm_backward");
  } else {
    const long long band = (rows + bands - 1) / bands;
    DISPATCH_IN(dtype, E, DISPATCH_FORMAT(format, F, {
      const LnKept<E> kept{static_cast<const E*>(x), mean, c, e, groups};
      const E* d = static_cast<const E*>(dy);
      if (dx) {
        launch(ln_dx_loop_kernel<E, F>, unsigned(std::min<long long>(rows, 148LL * 8)), LN_THREADS, 0, S(stream), d, kept, rstd,
               static_cast<const E*>(weight), static_cast<E*>(dx), rows, width);
        LAUNCH_CHECK("layer_norm_dx");
      }
      if (sums) {
        launch(ln_columns_kernel<E, F>, dim3(cdiv(width, 32), bands), 32 * COLUMN_LANES, 0, S(stream), d, kept, rstd, partials,
               rows, width, band);
        LAUNCH_CHECK("layer_norm_columns");
      }
    }));
  }
  if (sums) {
    DISPATCH_IN(dtype, E, (launch(column_fold_kernel<E>, dim3(cdiv(width, 32), 2), 32 * FOLD_LANES, 0, S(stream), partials,
                                  static_cast<E*>(dweight), static_cast<E*>(dbias), width, bands)));
    LAUNCH_CHECK("column_fold");
  }
  return 0;
}

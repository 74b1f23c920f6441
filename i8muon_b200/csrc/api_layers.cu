// C ABI: the layers around the stepped matrices (activations in eight bits, layer norm).
#include "host.cuh"
#include "layers.cuh"
#include "layer_passes.cuh"

using namespace i8m;

namespace i8m {

int eight_groups(int width) { return width / EIGHT_GROUP + (width % EIGHT_GROUP != 0); }

namespace {
unsigned eight_grid(long long groups) {
  return unsigned(std::min<long long>((groups + EIGHT_THREADS / 32 - 1) / (EIGHT_THREADS / 32), 148LL * 16));
}
}  // namespace

int eight_quant(const void* x, int dtype, long long rows, int width, int format, void* codes, void* exponents,
                cudaStream_t stream) {
  const int groups = eight_groups(width);
  const unsigned grid = eight_grid(rows * groups);
  uint8_t* c = static_cast<uint8_t*>(codes);
  uint8_t* e = static_cast<uint8_t*>(exponents);
  DISPATCH_IN(dtype, In, {
    auto kernel = format == EIGHT_INT8 ? eight_quant_kernel<In, EIGHT_INT8> : eight_quant_kernel<In, EIGHT_E4M3>;
    launch(kernel, grid, EIGHT_THREADS, 0, stream, static_cast<const In*>(x), c, e, rows, width, groups);
  });
  LAUNCH_CHECK("activation_quant");
  return 0;
}
int eight_restore(const void* codes, const void* exponents, long long rows, int width, int format, void* out, int dtype,
                  int pitch, cudaStream_t stream) {
  const int groups = eight_groups(width);
  const unsigned grid = eight_grid(rows * groups);
  const uint8_t* c = static_cast<const uint8_t*>(codes);
  const uint8_t* e = static_cast<const uint8_t*>(exponents);
  DISPATCH_IN(dtype, Out, {
    auto kernel = format == EIGHT_INT8 ? eight_restore_kernel<Out, EIGHT_INT8> : eight_restore_kernel<Out, EIGHT_E4M3>;
    launch(kernel, grid, EIGHT_THREADS, 0, stream, c, e, static_cast<Out*>(out), rows, width, groups, pitch);
  });
  LAUNCH_CHECK("activation_restore");
  return 0;
}

int pitch_rows(const void* src, void* dst, int dtype, long long rows, int width, int pitch, cudaStream_t stream) {
  const unsigned grid = unsigned(std::min<long long>((rows * (pitch / 8) + 255) / 256, 148LL * 16));
  if (dtype == I8M_F16)
    launch(pitch_rows_kernel<__half>, grid, 256, 0, stream, static_cast<const __half*>(src), static_cast<__half*>(dst), rows, width, pitch);
  else
    launch(pitch_rows_kernel<__nv_bfloat16>, grid, 256, 0, stream, static_cast<const __nv_bfloat16*>(src),
           static_cast<__nv_bfloat16*>(dst), rows, width, pitch);
  LAUNCH_CHECK("pitch_rows");
  return 0;
}

template <typename E>
static int linear_dz_typed(const LinearDz& d, cudaStream_t stream) {
  const int bands = row_bands(d.rows);
  const PreActivation<E> kept{static_cast<const E*>(d.z), static_cast<const uint8_t*>(d.codes),
                              static_cast<const uint8_t*>(d.exponents), d.z_pitch, eight_groups(d.width)};
  auto kernel = d.format == EIGHT_INT8 ? linear_dz_kernel<E, EIGHT_INT8>
              : d.format == EIGHT_E4M3 ? linear_dz_kernel<E, EIGHT_E4M3> : linear_dz_kernel<E, -1>;
  launch(kernel, dim3(cdiv(d.width, 32), bands), 32 * COLUMN_LANES, 0, stream, static_cast<const E*>(d.dy), kept,
         static_cast<E*>(d.dz), d.db ? d.partials : nullptr, d.rows, d.width, d.dz_pitch, (d.rows + bands - 1) / bands, d.activation);
  LAUNCH_CHECK("linear_dz");
  if (d.db) {
    launch(column_fold_kernel<E>, cdiv(d.width, 32), 32 * COLUMN_LANES, 0, stream, d.partials, static_cast<E*>(d.db),
           static_cast<E*>(nullptr), d.width, bands);
    LAUNCH_CHECK("column_fold");
  }
  return 0;
}
int linear_dz(const LinearDz& d, cudaStream_t stream) {
  return d.dtype == I8M_F16 ? linear_dz_typed<__half>(d, stream) : linear_dz_typed<__nv_bfloat16>(d, stream);
}

}  // namespace i8m

// ================================================================== eight-bit activations
static int check_eight(const char* name, const void* a, const void* codes, const void* exponents, long long rows, int width,
                       int dtype, int format) {
  if (!a || !codes || !exponents) return fail(I8M_E_ARGUMENT, "%s: null pointer", name);
  if (rows < 1 || width < 1) return fail(I8M_E_ARGUMENT, "%s: empty problem", name);
  if (!float_dtype_ok(dtype)) return fail(I8M_E_ARGUMENT, "%s: bad dtype %d", name, dtype);
  if (format != EIGHT_INT8 && format != EIGHT_E4M3) return fail(I8M_E_ARGUMENT, "%s: bad format %d", name, format);
  if (width > MAX_LAYER_WIDTH) return fail(I8M_E_LIMIT, "%s: width %d is above %d", name, width, MAX_LAYER_WIDTH);
  if (rows > MAX_LAYER_ROWS) return fail(I8M_E_LIMIT, "%s: %lld rows are above %lld", name, rows, MAX_LAYER_ROWS);
  return 0;
}
extern "C" int i8m_activation_quant(const void* x, int dtype, long long rows, int width, int format, void* codes,
                                    void* exponents, i8m_stream_t stream) {
  if (int rc = check_eight("activation_quant", x, codes, exponents, rows, width, dtype, format)) return rc;
  return eight_quant(x, dtype, rows, width, format, codes, exponents, S(stream));
}
extern "C" int i8m_activation_restore(const void* codes, const void* exponents, long long rows, int width, int format,
                                      void* out, int dtype, i8m_stream_t stream) {
  if (int rc = check_eight("activation_restore", out, codes, exponents, rows, width, dtype, format)) return rc;
  return eight_restore(codes, exponents, rows, width, format, out, dtype, width, S(stream));
}

// ================================================================== layer norm
namespace {

int check_norm(const char* name, const void* a, const void* b, long long rows, int width, int dtype, const void* codes,
               const void* exponents, int format) {
  if (!a || !b) return fail(I8M_E_ARGUMENT, "%s: null pointer", name);
  if (rows < 1 || width < 1) return fail(I8M_E_ARGUMENT, "%s: empty problem", name);
  if (!float_dtype_ok(dtype)) return fail(I8M_E_ARGUMENT, "%s: bad dtype %d", name, dtype);
  if (format < -1 || format > EIGHT_E4M3) return fail(I8M_E_ARGUMENT, "%s: bad format %d", name, format);
  if (format >= 0 && (!codes || !exponents)) return fail(I8M_E_ARGUMENT, "%s: null codes or exponents", name);
  if (width > MAX_LAYER_WIDTH) return fail(I8M_E_LIMIT, "%s: width %d is above %d", name, width, MAX_LAYER_WIDTH);
  if (rows > MAX_LAYER_ROWS) return fail(I8M_E_LIMIT, "%s: %lld rows are above %lld", name, rows, MAX_LAYER_ROWS);
  return 0;
}
#define DISPATCH_FORMAT(format, F, ...)                                       \
  do {                                                                        \
    if ((format) == EIGHT_INT8) { constexpr int F = EIGHT_INT8; __VA_ARGS__; } \
    else if ((format) == EIGHT_E4M3) { constexpr int F = EIGHT_E4M3; __VA_ARGS__; } \
    else { constexpr int F = -1; __VA_ARGS__; }                               \
  } while (0)
}  // namespace

extern "C" int i8m_layer_norm(const void* x, const void* weight, const void* bias, void* y, float* mean, float* rstd,
                              void* codes, void* exponents, int format, long long rows, int width, int dtype, float eps,
                              i8m_stream_t stream) {
  if (int rc = check_norm("layer_norm", x, y, rows, width, dtype, codes, exponents, format)) return rc;
  const int groups = eight_groups(width);
  const unsigned grid = unsigned(std::min<long long>(rows, 148LL * 8));
  DISPATCH_IN(dtype, E, DISPATCH_FORMAT(format, F, (launch(
      ln_forward_loop_kernel<E, F>, grid, LN_THREADS, 0, S(stream), static_cast<const E*>(x), static_cast<const E*>(weight),
      static_cast<const E*>(bias), static_cast<E*>(y), mean, rstd, static_cast<uint8_t*>(codes),
      static_cast<uint8_t*>(exponents), rows, width, groups, eps))));
  LAUNCH_CHECK("layer_norm");
  return 0;
}

extern "C" int i8m_layer_norm_scratch_bytes(long long rows, int width, size_t* bytes) {
  if (rows < 1 || width < 1 || !bytes) return fail(I8M_E_ARGUMENT, "layer_norm_scratch_bytes: bad argument");
  if (width > MAX_LAYER_WIDTH) return fail(I8M_E_LIMIT, "layer_norm_scratch_bytes: width %d is above %d", width, MAX_LAYER_WIDTH);
  *bytes = size_t(row_bands(rows)) * 2 * size_t(width) * sizeof(float);
  return 0;
}
extern "C" int i8m_layer_norm_backward(const void* dy, const void* x, const float* mean, const float* rstd, const void* codes,
                                       const void* exponents, int format, const void* weight, void* dx, void* dweight,
                                       void* dbias, long long rows, int width, int dtype, void* scratch, size_t scratch_bytes,
                                       i8m_stream_t stream) {
  if (int rc = check_norm("layer_norm_backward", dy, rstd, rows, width, dtype, codes, exponents, format)) return rc;
  if (format < 0 && (!x || !mean)) return fail(I8M_E_ARGUMENT, "layer_norm_backward: neither x and its means nor codes");
  if (!dx && !dweight && !dbias) return fail(I8M_E_ARGUMENT, "layer_norm_backward: nothing to compute");
  size_t need = 0;
  if (int rc = i8m_layer_norm_scratch_bytes(rows, width, &need)) return rc;
  const bool sums = dweight || dbias;
  if (sums && (!scratch || scratch_bytes < need))
    return fail(I8M_E_WORKSPACE, "layer_norm_backward: scratch %zu < %zu bytes", scratch ? scratch_bytes : 0, need);
  const int groups = eight_groups(width), bands = row_bands(rows);
  const long long band = (rows + bands - 1) / bands;
  float* partials = static_cast<float*>(scratch);
  DISPATCH_IN(dtype, E, DISPATCH_FORMAT(format, F, {
    const LnKept<E> kept{static_cast<const E*>(x), mean, static_cast<const uint8_t*>(codes),
                         static_cast<const uint8_t*>(exponents), groups};
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
  if (sums) {
    DISPATCH_IN(dtype, E, (launch(column_fold_kernel<E>, cdiv(width, 32), 32 * COLUMN_LANES, 0, S(stream), partials,
                                  static_cast<E*>(dweight), static_cast<E*>(dbias), width, bands)));
    LAUNCH_CHECK("column_fold");
  }
  return 0;
}

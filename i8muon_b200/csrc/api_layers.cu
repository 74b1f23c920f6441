// C ABI: the layers around the stepped matrices (activations in eight bits), and the passes of the linear layer.
#include "host.cuh"
#include "layers.cuh"
#include "layer_passes.cuh"

using namespace i8m;

namespace i8m {

int eight_groups(int width) { return width / EIGHT_GROUP + (width % EIGHT_GROUP != 0); }

namespace {
bool octets_fit(const void* p, int width, int pitch) {
  return width % EIGHT_GROUP == 0 && pitch == width && (reinterpret_cast<uintptr_t>(p) & 15u) == 0;
}
// Blocks of the list of octets (0: more than a launch has), and of the row kernels.
unsigned octet_blocks(long long octets) {
  const long long blocks = (octets + EIGHT_THREADS * EIGHT_UNROLL - 1) / (EIGHT_THREADS * EIGHT_UNROLL);
  return blocks <= 0x7fffffffLL ? unsigned(blocks) : 0;
}
// 16-bit rows of whole octets on 16 bytes take a kernel of their own (the workspace of a linear layer's backward pass).
template <typename Out, int FORMAT>
auto restore_rows(const void* out, int pitch) {
  auto kernel = eight_restore_rows_kernel<Out, FORMAT, false>;
  if constexpr (sizeof(Out) == 2) {
    if (pitch % 8 == 0 && on_octets(out, 2)) kernel = eight_restore_rows_kernel<Out, FORMAT, true>;
  }
  return kernel;
}
dim3 row_blocks(long long rows, int groups) {
  const unsigned segments = unsigned(cdiv(groups, EIGHT_SEGMENT));
  const long long most = std::max<long long>(1, 148LL * 32 / segments);
  return dim3(unsigned(std::min<long long>((rows + EIGHT_THREADS / 32 - 1) / (EIGHT_THREADS / 32), most)), segments);
}
}  // namespace

int eight_quant(const void* x, int dtype, long long rows, int width, int format, void* codes, void* exponents,
                cudaStream_t stream) {
  const int groups = eight_groups(width);
  const long long octets = rows * width / 8;
  uint8_t* c = static_cast<uint8_t*>(codes);
  uint8_t* e = static_cast<uint8_t*>(exponents);
  DISPATCH_IN(dtype, In, {
    const In* in = static_cast<const In*>(x);
    if (octets_fit(x, width, width) && octets_fit(codes, width, width) && octet_blocks(octets)) {
      auto kernel = format == EIGHT_INT8 ? eight_quant_octets_kernel<In, EIGHT_INT8> : eight_quant_octets_kernel<In, EIGHT_E4M3>;
      launch(kernel, octet_blocks(octets), EIGHT_THREADS, 0, stream, in, c, e, octets);
    } else {
      auto kernel = format == EIGHT_INT8 ? eight_quant_rows_kernel<In, EIGHT_INT8> : eight_quant_rows_kernel<In, EIGHT_E4M3>;
      launch(kernel, row_blocks(rows, groups), EIGHT_THREADS, 0, stream, in, c, e, rows, width, groups);
    }
  });
  LAUNCH_CHECK("activation_quant");
  return 0;
}
int eight_restore(const void* codes, const void* exponents, long long rows, int width, int format, void* out, int dtype,
                  int pitch, cudaStream_t stream) {
  const int groups = eight_groups(width);
  const long long octets = rows * width / 8;
  const uint8_t* c = static_cast<const uint8_t*>(codes);
  const uint8_t* e = static_cast<const uint8_t*>(exponents);
  DISPATCH_IN(dtype, Out, {
    Out* to = static_cast<Out*>(out);
    if (octets_fit(out, width, pitch) && on_octets(out, sizeof(Out)) && octets_fit(codes, width, width) && octet_blocks(octets)) {
      auto kernel = format == EIGHT_INT8 ? eight_restore_octets_kernel<Out, EIGHT_INT8> : eight_restore_octets_kernel<Out, EIGHT_E4M3>;
      launch(kernel, octet_blocks(octets), EIGHT_THREADS, 0, stream, c, e, to, octets);
    } else {
      auto kernel = format == EIGHT_INT8 ? restore_rows<Out, EIGHT_INT8>(out, pitch) : restore_rows<Out, EIGHT_E4M3>(out, pitch);
      launch(kernel, row_blocks(rows, groups), EIGHT_THREADS, 0, stream, c, e, to, rows, width, groups, pitch);
    }
  });
  LAUNCH_CHECK("activation_restore");
  return 0;
}

template <typename E>
static void launch_pitch_rows(const void* src0, void* dst0, long long rows0, const void* src1, void* dst1, long long rows1, int width,
                              int pitch, cudaStream_t stream) {
  const long long octets = ((dst0 ? rows0 : 0) + (dst1 ? rows1 : 0)) * (pitch / 8);
  launch(pitch_rows_kernel<E>, unsigned(std::min<long long>((octets + 255) / 256, 148LL * 16)), 256, 0, stream,
         static_cast<const E*>(src0), static_cast<E*>(dst0), rows0, static_cast<const E*>(src1), static_cast<E*>(dst1), rows1, width, pitch);
}
int pitch_rows(const void* src0, void* dst0, long long rows0, const void* src1, void* dst1, long long rows1, int dtype, int width,
               int pitch, cudaStream_t stream) {
  if (!dst0 && !dst1) return 0;
  if (dtype == I8M_F16) launch_pitch_rows<__half>(src0, dst0, rows0, src1, dst1, rows1, width, pitch, stream);
  else launch_pitch_rows<__nv_bfloat16>(src0, dst0, rows0, src1, dst1, rows1, width, pitch, stream);
  LAUNCH_CHECK("pitch_rows");
  return 0;
}

template <typename E>
static int linear_dz_typed(const LinearDz& d, cudaStream_t stream) {
  const int bands = dz_bands(d.rows, d.width);
  const long long band = (d.rows + bands - 1) / bands;
  const PreActivation<E> kept{static_cast<const E*>(d.z), static_cast<const uint8_t*>(d.codes),
                              static_cast<const uint8_t*>(d.exponents), d.z_pitch, eight_groups(d.width)};
  float* partials = d.db ? d.partials : nullptr;
  const bool aligned = d.width % 8 == 0 && on_octets(d.dy, 2);
  const bool active = d.activation != ACT_NONE;
  DISPATCH_FORMAT(active ? d.format : -1, F, {
    auto kernel = aligned ? linear_dz_kernel<E, F, true, true> : linear_dz_kernel<E, F, false, true>;
    if constexpr (F < 0)
      if (!active) kernel = aligned ? linear_dz_kernel<E, F, true, false> : linear_dz_kernel<E, F, false, false>;
    launch(kernel, dim3(cdiv(d.width, 256), bands), 32 * DZ_WARPS, 0, stream, static_cast<const E*>(d.dy), kept,
           static_cast<E*>(d.dz), partials, d.rows, d.width, d.dz_pitch, band, d.activation);
  });
  LAUNCH_CHECK("linear_dz");
  if (d.db) {
    launch(column_fold_kernel<E>, cdiv(d.width, 32), 32 * FOLD_LANES, 0, stream, d.partials, static_cast<E*>(d.db),
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
static int check_eight(const char* name, const void* a, const void* codes, const void* exponents, long long rows, long long width,
                       int dtype, int format) {
  if (!a || !codes || !exponents) return fail(I8M_E_ARGUMENT, "%s: null pointer", name);
  if (rows < 1 || width < 1) return fail(I8M_E_ARGUMENT, "%s: empty problem", name);
  if (!float_dtype_ok(dtype)) return fail(I8M_E_ARGUMENT, "%s: bad dtype %d", name, dtype);
  if (format != EIGHT_INT8 && format != EIGHT_E4M3) return fail(I8M_E_ARGUMENT, "%s: bad format %d", name, format);
  if (reinterpret_cast<uintptr_t>(codes) & 15u) return fail(I8M_E_ARGUMENT, "%s: codes are not 16-byte aligned", name);
  if (width > MAX_LAYER_WIDTH) return fail(I8M_E_LIMIT, "%s: width %lld is above %d", name, width, MAX_LAYER_WIDTH);
  if (rows > MAX_LAYER_ROWS) return fail(I8M_E_LIMIT, "%s: %lld rows are above %lld", name, rows, MAX_LAYER_ROWS);
  return 0;
}
extern "C" int i8m_activation_quant(const void* x, int dtype, long long rows, long long width, int format, void* codes,
                                    void* exponents, i8m_stream_t stream) {
  if (int rc = check_eight("activation_quant", x, codes, exponents, rows, width, dtype, format)) return rc;
  return eight_quant(x, dtype, rows, int(width), format, codes, exponents, S(stream));
}
extern "C" int i8m_activation_restore(const void* codes, const void* exponents, long long rows, long long width, int format,
                                      void* out, int dtype, i8m_stream_t stream) {
  if (int rc = check_eight("activation_restore", out, codes, exponents, rows, width, dtype, format)) return rc;
  return eight_restore(codes, exponents, rows, int(width), format, out, dtype, int(width), S(stream));
}

// What the translation units of the layer operators share on the host: limits and the passes that both call.
#pragma once
#include <cuda_runtime.h>

// The format as a constant: EIGHT_INT8, EIGHT_E4M3, or -1 for none.
#define DISPATCH_FORMAT(format, F, ...)                                       \
  do {                                                                        \
    if ((format) == EIGHT_INT8) { constexpr int F = EIGHT_INT8; __VA_ARGS__; } \
    else if ((format) == EIGHT_E4M3) { constexpr int F = EIGHT_E4M3; __VA_ARGS__; } \
    else { constexpr int F = -1; __VA_ARGS__; }                               \
  } while (0)

namespace i8m {

// Tensor-map coordinates and row counts of a launch are 32-bit; widths leave room for padding to 128.
constexpr int MAX_LAYER_WIDTH = 1 << 24;
constexpr long long MAX_LAYER_ROWS = 0x7fffffffLL - 1024;

// Bands that sums over rows are cut into: a function of the extents alone, because the order of a sum decides its bits.
constexpr int MAX_BANDS = 296;       // two blocks per SM
inline int row_bands(long long rows) { return int(rows < MAX_BANDS ? rows : MAX_BANDS); }

// Bands of a linear layer's bias gradient: enough blocks of 256 columns for eight per SM, 32 rows each at least.
inline int dz_bands(long long rows, int width) {
  const long long columns = (width + 255) / 256, wanted = (148LL * 8 + columns - 1) / columns, most = (rows + 31) / 32;
  const long long bands = wanted < most ? wanted : most;
  return int(bands < MAX_BANDS ? bands : MAX_BANDS);
}

// How a layer norm's rows are spread: `threads` per row (32: a warp, four rows to a block; otherwise a block) with `octets` of
// eight elements each, at most `most` (0: wider than the kernels that hold a row in registers).
constexpr int LN_FORWARD_OCTETS = 4, LN_BACKWARD_OCTETS = 2;
struct LnShape {
  int threads, octets;
  int block() const { return threads == 32 ? 128 : threads; }
  int rows_of_block() const { return threads == 32 ? 4 : 1; }
  // blocks that an SM holds at one time, by the threads that the registers allow and by shared memory
  int resident(int threads_of_sm, size_t smem) const {
    const int by_threads = threads_of_sm / block(), by_smem = int(227 * 1024 / (smem + 1024));
    const int n = by_threads < by_smem ? by_threads : by_smem;
    return n < 1 ? 1 : n;
  }
};
inline LnShape ln_shape(int width, int most) {
  const int octets = width / 8 + (width % 8 != 0);
  if (octets <= 32 * most) return {32, most == 2 && octets > 32 ? 2 : (octets + 31) / 32};
  // whole warps of threads; three octets instead of four where that leaves fewer idle (forward)
  auto threads = [&](int v) { return ((octets + v - 1) / v + 31) / 32 * 32; };
  if (most == 4 && threads(3) <= 512 && threads(3) * 3 < threads(4) * 4) return {threads(3), 3};
  for (int v = most; v <= 4; v *= 2)
    if (threads(v) <= 512) return {threads(v), v};
  return {0, 0};
}
// Bands of the backward pass's sums over rows, one per block of the register kernels: 512 resident threads per SM.
inline int ln_bands(long long rows, int width) {
  const LnShape s = ln_shape(width, LN_BACKWARD_OCTETS);
  if (!s.octets) return row_bands(rows);
  const long long blocks = (rows + s.rows_of_block() - 1) / s.rows_of_block(), most = 148LL * s.resident(512, 0);
  return int(blocks < most ? blocks : most);
}

// Whether octets of p (rows of whole octets) lie on their own size: what vectors are stored to.
inline bool on_octets(const void* p, size_t element) { return (reinterpret_cast<unsigned long long>(p) & (8 * element - 1)) == 0; }

int eight_groups(int width);
int eight_quant(const void* x, int dtype, long long rows, int width, int format, void* codes, void* exponents, cudaStream_t stream);
// out has `pitch` elements per row (width <= pitch <= 32 groups); those behind the width are written as zero
int eight_restore(const void* codes, const void* exponents, long long rows, int width, int format, void* out, int dtype, int pitch,
                  cudaStream_t stream);

// rows of `width` 16-bit elements copied to rows of `pitch`, of one or two matrices (a dst that is NULL is left out)
int pitch_rows(const void* src0, void* dst0, long long rows0, const void* src1, void* dst1, long long rows1, int dtype, int width,
               int pitch, cudaStream_t stream);
// dz = dy act'(z) into rows of dz_pitch (dz may be NULL), and db (may be NULL; partials: dz_bands x 2 x width floats)
struct LinearDz {
  const void* dy;
  const void* z;
  const void *codes, *exponents;
  int format, activation, dtype;
  long long rows;
  int width, z_pitch;
  void* dz;
  int dz_pitch;
  void* db;
  float* partials;
};
int linear_dz(const LinearDz& d, cudaStream_t stream);

}  // namespace i8m

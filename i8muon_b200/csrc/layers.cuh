// What the translation units of the layer operators share on the host: limits and the passes that both call.
#pragma once
#include <cuda_runtime.h>

namespace i8m {

// Tensor-map coordinates and row counts of a launch are 32-bit; widths leave room for padding to 128.
constexpr int MAX_LAYER_WIDTH = 1 << 24;
constexpr long long MAX_LAYER_ROWS = 0x7fffffffLL - 1024;

// Bands that sums over rows are cut into: a function of the rows alone, because the order of a sum decides its bits.
constexpr int MAX_BANDS = 296;       // two blocks per SM
inline int row_bands(long long rows) { return int(rows < MAX_BANDS ? rows : MAX_BANDS); }

int eight_groups(int width);
int eight_quant(const void* x, int dtype, long long rows, int width, int format, void* codes, void* exponents, cudaStream_t stream);
// out has `pitch` elements per row (width <= pitch <= 32 groups); those behind the width are written as zero
int eight_restore(const void* codes, const void* exponents, long long rows, int width, int format, void* out, int dtype, int pitch,
                  cudaStream_t stream);

// rows of `width` 16-bit elements copied to rows of `pitch`
int pitch_rows(const void* src, void* dst, int dtype, long long rows, int width, int pitch, cudaStream_t stream);
// dz = dy act'(z) into rows of dz_pitch (dz may be NULL), and db (may be NULL; partials: row_bands(rows) x 2 x width floats)
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

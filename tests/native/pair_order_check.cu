// Host-side check of the unit order of linear_pair_kernel: every 256 x 256 unit of a product exactly once, inside the matrix.
// Compiled by tests/test_pair_order.py with nvcc as plain host code; prints "ok" or the first violation.
#include <cstdio>
#include <vector>
#include "gemm_linear_pair.cuh"

using namespace i8m;

int main() {
  const int groups[] = {8, 10, 16, 32, 64};
  for (int group : groups)
    for (int m = 1; m <= 150; ++m)
      for (int n = 1; n <= 70; ++n) {
        GemmGeom g{};
        g.tiles_m = m; g.tiles_n = n; g.group = group;
        const int rows = (m + 1) / 2, cols = (n + 1) / 2;
        std::vector<char> seen(size_t(rows) * cols, 0);
        for (int u = 0; u < rows * cols; ++u) {
          int r = -1, c = -1;
          decode_pair(g, u, r, c);
          if (r < 0 || r >= rows || c < 0 || c >= cols || seen[size_t(r) * cols + c]++)
            return std::printf("m%d n%d group %d unit %d -> (%d, %d)\n", m, n, group, u, r, c);
        }
      }
  // cut along K: every K block of every unit in exactly one part, in order
  for (int kb : {4, 5, 17, 256, 1025})
    for (int parts = 1; parts <= 64 && parts <= kb; ++parts)
      for (int m = 1; m <= 9; ++m) {
        GemmGeom g{};
        g.tiles_m = m; g.tiles_n = 3; g.group = 8; g.num_kb = kb;
        const int units = (m + 1) / 2 * 2;
        for (int u = 0; u < units; ++u)
          for (int p = 0, at = 0; p < parts; ++p) {
            const PairItem it = decode_item<true>(g, parts, u * parts + p);
            int r, c;
            decode_pair(g, u, r, c);
            if (it.part != p || it.row_pair != r || it.col_pair != c || it.kb0 != at || it.kb1 <= at || (p == parts - 1 && it.kb1 != kb))
              return std::printf("kb %d parts %d m%d unit %d part %d -> (%d, %d) %d [%d, %d)\n", kb, parts, m, u, p, it.row_pair, it.col_pair,
                                 it.part, it.kb0, it.kb1);
            at = it.kb1;
          }
      }
  std::puts("ok");
  return 0;
}

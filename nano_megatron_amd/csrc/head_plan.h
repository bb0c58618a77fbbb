// The tiles of the LM head's products whose epilogue is a loss (head.hip, distill.hip).
#pragma once

#include <stdint.h>

namespace nmb {
namespace {

// Tiles of a launch.  64 x 64 ones where there are at most four a CU (or no more rows than
// that): all are under way at once, and the more workgroups bring the table in faster; then
// 128 x 256 while there is at most one a CU; else 256 x 256, and 256 x 128 in the backward,
// whose two workgroups a CU overlap one's epilogue, longer than the forward's, with the
// other's products.  us, forward / gradient, the tiles taken first:
//   128 x 8192 x 768:    64 x 64 9.6 / 6.7, 128 x 256 18.3 / 17.4, 256 x 256 25.8 / 26.6
//   256 x 32000 x 768:   128 x 256 23.0 / 22.0, 64 x 64 31.5 / 27.6, 256 x 256 29.3 / 30.0
//   1024 x 8192 x 768:   128 x 256 20.1 / 21.3, 64 x 64 30.0 / 28.1, 256 x 256 26.8 / 30.2
//   2048 x 50304 x 768:  256 x 256 182, 128 x 256 206 / 256 x 128 194, 256 x 256 213
//   8192 x 50304 x 768:  256 x 256 638, 128 x 256 760 / 256 x 128 780, 256 x 256 893
struct HeadPlan {
  int tbm, tbn;
};
HeadPlan head_plan(int64_t rows, int64_t vocab, bool backward) {
  auto tiles = [&](int64_t m, int64_t n) { return (rows + m - 1) / m * ((vocab + n - 1) / n); };
  if (rows <= 64 || tiles(64, 64) <= 4 * 256) return HeadPlan{64, 64};
  if (rows <= 128 || tiles(128, 256) <= 256) return HeadPlan{128, 256};
  return HeadPlan{256, backward ? 128 : 256};
}

int64_t head_tiles_n(int64_t rows, int64_t vocab) {  // of the forward
  const HeadPlan p = head_plan(rows, vocab, false);
  return (vocab + p.tbn - 1) / p.tbn;
}

}  // namespace
}  // namespace nmb

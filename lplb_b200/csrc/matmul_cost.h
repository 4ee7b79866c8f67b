// What the launches of a product are chosen by.  Plain C++, in 64 bits: k goes up to 2^28 and the rows up to 2^31.
#pragma once

#include <stdint.h>

namespace lplb {
namespace ops {

// What a product takes, in cycles beside the launch: an SM is fed by some 64 bytes a cycle from the L2 and computes a block of 64 of 256
// features x n rows (a pair) in 2 n cycles; then the last tile's way out.
inline int64_t block_cycles(int64_t n) { return n < 256 ? 256 + n : 2 * n; }
// One group: result rows in tiles of equal height, so high that this is least over the rounds of CTA pairs.  Several groups: their
// rows are only known on the device.
struct PairCost {
  int64_t cycles;
  int steps;  // of a tile
};
inline PairCost pair_cost(int64_t rows, int step, int most_rows, int64_t tiles_p, int64_t k_blocks, int n_sm) {
  const int64_t steps = (rows + step - 1) / step;
  PairCost best{INT64_MAX, most_rows / step};
  for (int s = most_rows / step; s >= 1; --s) {
    const int64_t tiles = (steps + s - 1) / s, high = (steps + tiles - 1) / tiles, n = high * step;
    const int64_t rounds = (tiles * tiles_p + n_sm / 2 - 1) / (n_sm / 2), cycles = rounds * (k_blocks * block_cycles(n) + 100) + 8 * n;
    if (cycles < best.cycles) best = {cycles, (int)high};
  }
  return best;
}

// Few rows: `tiles` of 128 rows of b times `cols` rows of a, `fit` of them at once, each of `split` CTAs with `blocks` k blocks.
inline int64_t few_cycles(int64_t tiles, int64_t fit, int64_t blocks, int64_t cols, int split) {
  return (tiles + fit - 1) / fit * (blocks * (256 + 2 * cols) + 10 * cols + (split > 1 ? 1500 + 2 * cols : 0));
}

}  // namespace ops
}  // namespace lplb

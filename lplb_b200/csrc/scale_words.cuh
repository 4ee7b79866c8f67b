// Scales of operands in 8 bits on their way to tensor memory.
#pragma once

#include <stdint.h>

namespace lplb {
namespace ops {

constexpr uint32_t kScaleAtom = 512;         // scales of 128 rows and 4 blocks in shared memory
constexpr uint32_t kScaleOnes = 0x7F7F7F7F;  // four scales of 1

// Scales are fetched 16 blocks at a time and one such chunk ahead: an ordinary load waits behind
// the operands that TMA has under way to the same SM, several microseconds where those are 200 KB.  All loads of a chunk
// go out together, so nothing is asked in between: what lies behind a row's last block is never used, and loads that
// would start there read the last block's word again.
constexpr int kScaleChunk = 16;
struct ScaleChunk {
  uint32_t word[4];
  // blocks 16 * chunk ... of a row of k_blocks scales.  WORDS: rows start on 4-byte boundaries and k_blocks is a multiple of 4.
  template <bool WORDS>
  __device__ __forceinline__ void fetch(const uint8_t* row, int chunk, int k_blocks) {
    const uintptr_t p = reinterpret_cast<uintptr_t>(row) + kScaleChunk * chunk;
    const uintptr_t last = (reinterpret_cast<uintptr_t>(row) + k_blocks - 1) & ~(uintptr_t)3;  // word that holds the last block
    if constexpr (WORDS) {
#pragma unroll
      for (int i = 0; i < 4; ++i) word[i] = __ldcg(reinterpret_cast<const uint32_t*>(min(p + 4 * i, last)));
    } else {
      uint32_t w[5];
#pragma unroll
      for (int i = 0; i < 5; ++i) w[i] = __ldcg(reinterpret_cast<const uint32_t*>(min((p & ~(uintptr_t)3) + 4 * i, last)));
#pragma unroll
      for (int i = 0; i < 4; ++i) word[i] = __funnelshift_r(w[i], w[i + 1], 8 * (uint32_t)(p & 3));
    }
  }
};

}  // namespace ops
}  // namespace lplb

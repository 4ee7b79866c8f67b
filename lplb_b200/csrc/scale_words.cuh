// Scales of operands in 8 bits on their way to tensor memory.
#pragma once

#include <stdint.h>

namespace lplb {
namespace ops {

constexpr uint32_t kScaleAtom = 512;         // scales of 128 rows and 4 blocks in shared memory
constexpr uint32_t kScaleOnes = 0x7F7F7F7F;  // four scales of 1

// Four scale bytes of blocks 4 * group ... of a row, 1 beyond the last block.
__device__ __forceinline__ uint32_t scale_word(const uint8_t* row, int group, int k_blocks, bool words) {
  if (words) return __ldcg(reinterpret_cast<const uint32_t*>(row) + group);
  uint32_t w = kScaleOnes;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (4 * group + i < k_blocks) w = (w & ~(0xFFu << (8 * i))) | ((uint32_t)__ldcg(row + 4 * group + i) << (8 * i));
  return w;
}

// Scales are fetched 16 blocks at a time and one such chunk ahead: an ordinary load waits behind
// the operands that TMA has under way to the same SM, several microseconds where those are 200 KB.
constexpr int kScaleChunk = 16;
struct ScaleChunk {
  uint32_t word[4];
  // blocks 16 * chunk ... of a row; `on`: else ones
  __device__ __forceinline__ void fetch(const uint8_t* row, int chunk, int k_blocks, bool words, bool on) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      word[i] = on && kScaleChunk * chunk + 4 * i < k_blocks ? scale_word(row, 4 * chunk + i, k_blocks, words) : kScaleOnes;
  }
};

}  // namespace ops
}  // namespace lplb

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

}  // namespace ops
}  // namespace lplb

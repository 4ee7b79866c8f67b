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
template <bool WORDS>  // rows start on 4-byte boundaries and k_blocks is a multiple of 4
struct ScaleChunk {
  uint32_t raw[WORDS ? 4 : 5];
  uint32_t shift;
  // blocks 16 * chunk ... of a row of k_blocks scales
  __device__ __forceinline__ void fetch(const uint8_t* row, int chunk, int k_blocks) {
    const uintptr_t p = reinterpret_cast<uintptr_t>(row) + kScaleChunk * chunk;
    const uintptr_t last = (reinterpret_cast<uintptr_t>(row) + k_blocks - 1) & ~(uintptr_t)3;  // word that holds the last block
    shift = 8 * (uint32_t)(p & 3);
#pragma unroll
    for (int i = 0; i < (WORDS ? 4 : 5); ++i) raw[i] = __ldcg(reinterpret_cast<const uint32_t*>(min((p & ~(uintptr_t)3) + 4 * i, last)));
  }
  // blocks 4 * i ... of the chunk: put together here, where the loads have to be there anyway
  __device__ __forceinline__ uint32_t word(int i) const {
    if constexpr (WORDS) return raw[i];
    else return __funnelshift_r(raw[i], raw[i + 1], shift);
  }
};

}  // namespace ops
}  // namespace lplb

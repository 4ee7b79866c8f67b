// The forward product in 16 bits for few rows, or small: z = a b^T + bias, out = act(z) + residual.
//
// Bound by reading b once.  A CTA computes 128 rows of b against all rows of a (or a part of them, where b is small): the weights on the
// tensor core's M side, so that few rows cost few cycles, and the k blocks of a tile are dealt out to the CTAs of a cluster, so
// that a matrix with few tiles still occupies every SM.  The partial sums meet in distributed shared memory, in rank order: no
// workspace, nothing to clear, the same bits every time; the epilogue comes after the sum.
//
// Roles (256 threads): warp 0 TMA, warp 1 matrix instructions, warps 4-7 tensor memory to shared memory; all of them add up the
// partial sums and finish.
#pragma once

#include "matmul.cuh"

namespace lplb {
namespace ops {

constexpr int kFewTileRows = 128, kFewKBytes = 128, kFewStageMax = 12, kFewBlock = 256, kFewMostRows = 256, kFewMostSplit = 8;
constexpr uint32_t kFewWeightStage = kFewTileRows * kFewKBytes;
constexpr uint32_t kFewSmemPerColumn = 448;  // of 228 KB, 1 KB of them per CTA: columns, powers of two from 64, add up to 512 at most

struct FewProductArgs {
  int* status;
  unsigned long long budget_ns;
  int m, k_blocks;
  int tiles;   // of 128 rows of b
  int cols;    // rows of a per CTA, a multiple of 16
  int chains;  // accumulators, of consecutive k blocks each: a result in 32 bits is summed in parts (kSumBlocks)
  int stages;
  int wide;    // as PairArgs
  uint32_t idesc;
  Epilogue e;
};

// Shared memory from a 1024-byte boundary on.  A launch asks for `request` bytes: at least as large a part of an SM's shared memory as its
// columns are of the tensor memory, so that CTAs that are on an SM together always find their columns free.
struct FewProductLayout {
  uint32_t stage, bars, total, columns, request;
  __host__ __device__ FewProductLayout(int cols, int chains, int stages) {
    stage = kFewWeightStage + cols * kFewKBytes;
    bars = stage * stages;
    const uint32_t partial = (uint32_t)cols * kFewTileRows * 4;  // over the ring, once it has been read
    if (bars < partial) bars = partial;
    total = bars + (2 * kFewStageMax + 1) * 8;
    columns = cols * chains <= 64 ? 64 : cols * chains <= 128 ? 128 : 256;
    request = total + 1024 > columns * kFewSmemPerColumn ? total + 1024 : columns * kFewSmemPerColumn;
  }
};

template <bool GATED>
__global__ void __launch_bounds__(kFewBlock, 1)
few_product_kernel(const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_a, const FewProductArgs a) {
  using namespace sm100;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const FewProductLayout at(a.cols, a.chains, a.stages);
  const uint32_t base = smem_u32(smem);
  const uint32_t bar_full = base + at.bars, bar_empty = bar_full + 8 * kFewStageMax, bar_done = bar_empty + 8 * kFewStageMax;
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cluster_cta_rank(), split = (int)cluster_size();
  const int tile = (int)blockIdx.x / split % a.tiles, m0 = (int)blockIdx.x / split / a.tiles * a.cols, m_here = min(a.cols, a.m - m0);
  const int kb0 = (int)((int64_t)a.k_blocks * rank / split), kb1 = (int)((int64_t)a.k_blocks * (rank + 1) / split);
  const int per_chain = (kb1 - kb0 + a.chains - 1) / a.chains;  // k blocks
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < kFewStageMax; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    mbar_init(bar_done, 1);
    fence_barrier_init();
    tma_prefetch_desc(&map_a);
    tma_prefetch_desc(&map_b);
  }
  if (warp == 1) tmem_alloc_single(smem_u32(&tmem_slot), at.columns);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = tmem_slot;
  volatile int* abort = &abort_flag;
  wait_predecessors();
  allow_successor();

  if (warp == 0) {
    if (elect_one()) {
      uint32_t s = 0, ph = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(bar_empty + 8 * s, ph ^ 1, abort, a.budget_ns)) break;
        const uint32_t dst = base + s * at.stage;
        mbar_expect_tx(bar_full + 8 * s, at.stage);
        if constexpr (GATED) {  // 64 gate rows, their 64 up rows
          const int gate = tile / 2 * (2 * kGateBlock) + tile % 2 * (kGateBlock / 2);
          tma_load_2d(dst, &map_b, bar_full + 8 * s, kb * kPairK, gate);
          tma_load_2d(dst + kFewWeightStage / 2, &map_b, bar_full + 8 * s, kb * kPairK, gate + kGateBlock);
        } else {
          tma_load_2d(dst, &map_b, bar_full + 8 * s, kb * kPairK, tile * kFewTileRows);
        }
        tma_load_2d(dst + kFewWeightStage, &map_a, bar_full + 8 * s, kb * kPairK, m0);
        if (++s == (uint32_t)a.stages) s = 0, ph ^= 1;
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      const uint32_t idesc = a.idesc | umma_idesc_size(kFewTileRows, a.cols);
      uint32_t s = 0, ph = 0;
      uint32_t tmem_d = tmem - a.cols;
      for (int kb = kb0, in_chain = 0; kb < kb1; ++kb, in_chain = in_chain + 1 < per_chain ? in_chain + 1 : 0) {
        if (!mbar_wait(bar_full + 8 * s, ph, abort, a.budget_ns)) break;
        tc_fence_after_sync();
        if (in_chain == 0) tmem_d += a.cols;
        const uint32_t src = base + s * at.stage;
        const uint64_t dw = umma_desc_sw128(src), dt = umma_desc_sw128(src + kFewWeightStage);
#pragma unroll
        for (int k = 0; k < kPairK / 16; ++k) umma_bf16(tmem_d, dw + 2 * k, dt + 2 * k, idesc, in_chain != 0 || k != 0);
        umma_commit(bar_empty + 8 * s);
        if (++s == (uint32_t)a.stages) s = 0, ph ^= 1;
      }
      umma_commit(bar_done);
    }
  } else if (warp >= 4) {
    const bool done = mbar_wait(bar_done, 0, abort, a.budget_ns);
    __syncwarp();
    if (__all_sync(0xffffffffu, done)) {
      tc_fence_after_sync();
      const int row = (warp & 3) * 32 + lane;
      float* partial = reinterpret_cast<float*>(smem);
      for (int c0 = 0; c0 < a.cols; c0 += 16) {
        float v[16];
        tmem_ld_32x16(tmem + ((uint32_t)((warp & 3) * 32) << 16) + c0, v);
        tmem_ld_wait();
        for (int chain = 1; chain * per_chain < kb1 - kb0; ++chain) {
          float more[16];
          tmem_ld_32x16(tmem + ((uint32_t)((warp & 3) * 32) << 16) + chain * a.cols + c0, more);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; ++i) v[i] += more[i];
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) partial[(c0 + i) * kFewTileRows + row] = v[i];
      }
      tc_fence_before_sync();
    }
  }
  __syncthreads();
  if (*abort) {  // a role gave up: copies in flight land before shared memory and tensor memory are released
    const uint64_t t0 = timer_ns();
    while (timer_ns() - t0 < 200000) __nanosleep(1000);
    if (threadIdx.x == 0) atomicCAS(a.status, 0, (int)kOpsTimeout);
  }
  // The accumulators have been read: no CTA holds columns while it waits for its cluster, whatever else is on its SM.
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc_single(tmem, at.columns);
  }
  if (split > 1) cluster_sync();
  // The CTAs share a tile's rows of a out among their threads, four columns of the result to each.
  auto join = [&](auto wide) {
    constexpr bool kWide = decltype(wide)::value;
    constexpr int kLanes = GATED ? 16 : 32, S = kWide ? 1 : kLanes;
    const int in_row = threadIdx.x & (kLanes - 1), f = kWide ? 4 * in_row : in_row;
    Columns<S, GATED> mine;
    if constexpr (GATED) {
      mine.out = tile * (kFewTileRows / 2) + f;
      mine.gate = tile / 2 * (2 * kGateBlock) + tile % 2 * (kGateBlock / 2) + f;
      mine.limit = kFewTileRows;  // whole blocks
    } else {
      mine.out = mine.gate = tile * kFewTileRows + f;
      mine.limit = a.e.n - mine.out;
    }
    mine.load_bias(a.e, 0);
    for (int i = rank * kFewBlock + threadIdx.x; i < m_here * kLanes; i += split * kFewBlock) {
      const int m = i / kLanes;
      float z[4] = {}, up[4] = {}, r[4];
      mine.load_residual(a.e, m0 + m, r);
      for (int other = 0; other < split; ++other) {
        const uint32_t from = map_to_rank(base + (uint32_t)(m * kFewTileRows + f) * 4, other);
        auto add = [&](uint32_t where, float (&to)[4]) {
          if constexpr (kWide) {
            const float4 v = ld_cluster_v4(where);
            to[0] += v.x, to[1] += v.y, to[2] += v.z, to[3] += v.w;
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) to[j] += ld_cluster_f32(where + j * S * 4);
          }
        };
        add(from, z);
        if (GATED) add(from + kFewTileRows / 2 * 4, up);
      }
      mine.finish(a.e, m0 + m, z, up, r);
    }
  };
  if (a.wide) join(std::true_type{});
  else join(std::false_type{});
  if (split > 1) cluster_sync();  // no CTA leaves while another reads its sums
}

}  // namespace ops
}  // namespace lplb

// C[m, n] = sum over blocks of 128 along k of sa[m, kb] * sb[n / 128, kb] * sum_k A[m, k] * B[n, k]
// for few rows m, or small products: e4m3 operands, power-of-two scales that the tensor cores multiply in by themselves.
//
// Bound by reading B once.  A CTA computes 128 rows of B against all rows of A (or a part of them, where B is small): the weights
// on the tensor core's M side, so that few rows cost few cycles, and the k blocks of a tile are dealt out to the CTAs of a
// cluster, so that a matrix with few tiles still occupies every SM.  The partial sums meet in distributed shared
// memory, in rank order: no workspace, nothing to clear, the same bits every time.  64 x 4096 x 7168 (29.8 MB) take
// 10.4 us among others, 2.9 TB/s; 1 x 7168 x 2048 5.4 us: launch, the first load and the join are half of it.
//
// Roles (256 threads): warp 0 TMA producer, warp 1 matrix instructions, warp 2 scales, warps 4-7
// epilogue; all of them add up the partial sums.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>

#include <type_traits>

#include "common.cuh"
#include "ops_api.h"
#include "scale_words.cuh"
#include "tcgen05.cuh"

namespace lplb {
namespace ops {

constexpr int kTileRows = 128;                  // weight rows per CTA
constexpr int kKBytes = 128;                    // bytes of a row per k block
constexpr uint32_t kWeightStage = kTileRows * kKBytes;
constexpr int kMaxRingStages = 12;
constexpr int kScaleSlots = 4;
constexpr int kFewThreads = 256;
constexpr int kFewMaxRows = 256;                // of A per CTA
constexpr int kMaxSplit = 8;                    // portable cluster size
constexpr uint32_t kSmemPerColumn = 448;        // of 228 KB, 1 KB of them per CTA: columns, multiples of 64, add up to 512 at most

struct FewArgs {
  const uint8_t* a_scale;  // [m, a_scale_ld]
  const uint8_t* b_scale;  // [ceil(n / 128), k_blocks]
  void* out;               // [m, out_ld]
  int* error;              // the device's error word
  unsigned long long budget_ns;
  int64_t a_scale_ld, out_ld;
  int m, n, k_blocks;
  int tiles;               // of 128 rows of B
  int cols;                // rows of A per CTA, a multiple of 16
  int stages;
  int scale_words;         // scale rows start on 4-byte boundaries
};

// Shared memory from a 1024-byte boundary on.  A launch asks for `request` bytes: at least as large a part of an SM's shared
// memory as its columns are of the tensor memory, so that CTAs that are on an SM together (of this kernel, any size,
// any stream) always find their columns free.  Columns are given back before a CTA waits for its cluster: one that has to wait
// for another kernel's columns all the same is late, and holds nothing up.
struct FewLayout {
  uint32_t stage, ring, scales, bars, total, columns, request;
  __host__ __device__ FewLayout(int cols, int stages) {
    stage = kWeightStage + cols * kKBytes;
    ring = 0;
    scales = stage * stages;
    const uint32_t partial = (uint32_t)cols * kTileRows * 4;  // over the ring, once it has been read
    if (scales < partial) scales = partial;
    bars = scales + kScaleSlots * 3 * kScaleAtom;
    total = bars + (2 * kMaxRingStages + 2 * kScaleSlots + 1) * 8;
    const uint32_t used = scale_columns(cols) + 16;
    columns = used <= 64 ? 64 : used <= 128 ? 128 : used <= 256 ? 256 : 512;
    request = total + 1024 > columns * kSmemPerColumn ? total + 1024 : columns * kSmemPerColumn;
  }
  static __host__ __device__ uint32_t scale_columns(int cols) { return (uint32_t)(cols + 31) / 32 * 32; }  // where the scales begin
};

__device__ __forceinline__ void store_out(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_out(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

template <typename Out>
__global__ void __launch_bounds__(kFewThreads, 1)
few_rows_kernel(const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_a, const FewArgs a) {
  using namespace sm100;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const FewLayout at(a.cols, a.stages);
  const uint32_t base = smem_u32(smem), bars = base + at.bars;
  const uint32_t bar_full = bars, bar_empty = bars + 8 * kMaxRingStages;
  const uint32_t bar_sfull = bars + 16 * kMaxRingStages, bar_sempty = bar_sfull + 8 * kScaleSlots;
  const uint32_t bar_done = bar_sempty + 8 * kScaleSlots;
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cluster_cta_rank(), split = (int)(cluster_size());
  const int tile = (int)blockIdx.x / split % a.tiles, m0 = (int)blockIdx.x / split / a.tiles * a.cols, m_here = min(a.cols, a.m - m0);
  const int kb0 = (int)((int64_t)a.k_blocks * rank / split), kb1 = (int)((int64_t)a.k_blocks * (rank + 1) / split);
  const uint32_t scale_cols = FewLayout::scale_columns(a.cols), tmem_cols = at.columns;
  allow_successor();
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < kMaxRingStages; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    for (int s = 0; s < kScaleSlots; ++s) {
      mbar_init(bar_sfull + 8 * s, 1);
      mbar_init(bar_sempty + 8 * s, 1);
    }
    mbar_init(bar_done, 1);
    fence_barrier_init();
    tma_prefetch_desc(&map_a);
    tma_prefetch_desc(&map_b);
  }
  if (warp == 1) tmem_alloc_single(smem_u32(&tmem_slot), tmem_cols);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = tmem_slot;
  volatile int* abort = &abort_flag;
  wait_predecessors();

  if (warp == 0) {
    if (elect_one()) {
      uint32_t s = 0, ph = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(bar_empty + 8 * s, ph ^ 1, abort, a.budget_ns)) break;
        const uint32_t dst = base + s * at.stage;
        mbar_expect_tx(bar_full + 8 * s, at.stage);
        tma_load_2d(dst, &map_b, bar_full + 8 * s, kb * kKBytes, tile * kTileRows);
        tma_load_2d(dst + kWeightStage, &map_a, bar_full + 8 * s, kb * kKBytes, m0);
        if (++s == (uint32_t)a.stages) s = 0, ph ^= 1;
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      const uint32_t idesc = umma_idesc_mxf8(kTileRows, a.cols);
      const uint32_t tmem_sa = tmem + scale_cols, tmem_sb = tmem_sa + 4;
      uint32_t s = 0, ph = 0, ss = 0, sph = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (kb == kb0 || (kb & 3) == 0) {
          if (!mbar_wait(bar_sfull + 8 * ss, sph, abort, a.budget_ns)) break;
          tc_fence_after_sync();
          const uint32_t src = base + at.scales + ss * 3 * kScaleAtom;
          tmem_cp_scales(tmem_sa, src);
          for (int i = 0; i * 128 < a.cols; ++i) tmem_cp_scales(tmem_sb + 4 * i, src + (1 + i) * kScaleAtom);
          umma_commit(bar_sempty + 8 * ss);
          if (++ss == kScaleSlots) ss = 0, sph ^= 1;
        }
        if (!mbar_wait(bar_full + 8 * s, ph, abort, a.budget_ns)) break;
        tc_fence_after_sync();
        const uint32_t src = base + s * at.stage;
        const uint64_t dw = umma_desc_sw128(src), dt = umma_desc_sw128(src + kWeightStage);
        const uint32_t id = umma_idesc_scale_byte(idesc, kb & 3);
#pragma unroll
        for (int k = 0; k < 4; ++k)  // 32 values = 32 bytes along k inside the swizzled row
          umma_mxf8(tmem, dw + 2 * k, dt + 2 * k, id, tmem_sa, tmem_sb, kb != kb0 || k != 0);
        umma_commit(bar_empty + 8 * s);
        if (++s == (uint32_t)a.stages) s = 0, ph ^= 1;
      }
      umma_commit(bar_done);
    }
  } else if (warp == 2) {
    const uint8_t* b_row = a.b_scale + (int64_t)tile * a.k_blocks;
    uint32_t ss = 0, sph = 0;
    auto stage = [&](auto words) {
      ScaleChunk<decltype(words)::value> next[9], now[9];
      auto fetch = [&](int chunk) {
#pragma unroll
        for (int j = 0; j < 8; ++j)  // a row that is not there has a column that nobody reads
          if (j == 0 || 32 * j < a.cols) next[j].fetch(a.a_scale + (int64_t)(m0 + min(lane + 32 * j, m_here - 1)) * a.a_scale_ld, chunk, a.k_blocks);
        next[8].fetch(b_row, chunk, a.k_blocks);
      };
      const int last = (kb1 - 1) / kScaleChunk;
      fetch(kb0 / kScaleChunk);
      for (int chunk = kb0 / kScaleChunk; chunk <= last; ++chunk) {
#pragma unroll
        for (int j = 0; j < 9; ++j) now[j] = next[j];
        if (chunk < last) fetch(chunk + 1);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int kb = chunk * kScaleChunk + 4 * i;
          if (kb + 4 <= kb0 || kb >= kb1) continue;
          if (!__all_sync(0xffffffffu, mbar_wait(bar_sempty + 8 * ss, sph ^ 1, abort, a.budget_ns))) return;
          const uint32_t w = now[8].word(i);
          uint8_t* dst = smem + at.scales + ss * 3 * kScaleAtom + lane * 16;
          *reinterpret_cast<uint4*>(dst) = make_uint4(w, w, w, w);
          *reinterpret_cast<uint4*>(dst + kScaleAtom) = make_uint4(now[0].word(i), now[1].word(i), now[2].word(i), now[3].word(i));
          if (a.cols > 128)
            *reinterpret_cast<uint4*>(dst + 2 * kScaleAtom) = make_uint4(now[4].word(i), now[5].word(i), now[6].word(i), now[7].word(i));
          fence_proxy_async_shared();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar_sfull + 8 * ss);
          if (++ss == kScaleSlots) ss = 0, sph ^= 1;
        }
      }
    };
    if (a.scale_words) stage(std::true_type{});
    else stage(std::false_type{});
  } else if (warp >= 4) {
    const bool done = mbar_wait(bar_done, 0, abort, a.budget_ns);
    __syncwarp();
    if (__all_sync(0xffffffffu, done)) {
      tc_fence_after_sync();
      const int row = (warp & 3) * 32 + lane, n = tile * kTileRows + row;
      float* partial = reinterpret_cast<float*>(smem);
      for (int c0 = 0; c0 < a.cols; c0 += 16) {
        float v[16];
        tmem_ld_32x16(tmem + ((uint32_t)((warp & 3) * 32) << 16) + c0, v);
        tmem_ld_wait();
        if (split > 1) {
#pragma unroll
          for (int i = 0; i < 16; ++i) partial[(c0 + i) * kTileRows + row] = v[i];
        } else if (n < a.n) {
          Out* out = static_cast<Out*>(a.out) + (int64_t)(m0 + c0) * a.out_ld + n;
#pragma unroll
          for (int i = 0; i < 16; ++i, out += a.out_ld)
            if (c0 + i < m_here) store_out(out, v[i]);
        }
      }
      tc_fence_before_sync();
    }
  }
  __syncthreads();
  if (*abort) {  // a role gave up: copies in flight land before shared memory and tensor memory are released
    const uint64_t t0 = timer_ns();
    while (timer_ns() - t0 < 200000) __nanosleep(1000);
    if (threadIdx.x == 0) atomicCAS(a.error, 0, kOpsTimeout);
  }
  // The accumulators have been read: no CTA holds columns while it waits for its cluster, whatever else is on its SM.
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc_single(tmem, tmem_cols);
  }
  if (split > 1) {
    cluster_sync();
    // 128 sums of a row of A are 32 x 4; the CTAs share the rows out among their threads
    for (int i = rank * kFewThreads + threadIdx.x; i < m_here * 32; i += split * kFewThreads) {
      const int m = i >> 5, c = (i & 31) * 4, n = tile * kTileRows + c;
      const uint32_t mine = base + (uint32_t)i * 16;
      float4 sum = ld_cluster_v4(map_to_rank(mine, 0));
      for (int r = 1; r < split; ++r) {
        const float4 f = ld_cluster_v4(map_to_rank(mine, r));
        sum.x += f.x, sum.y += f.y, sum.z += f.z, sum.w += f.w;
      }
      Out* out = static_cast<Out*>(a.out) + (int64_t)(m0 + m) * a.out_ld + n;
      if (n < a.n) store_out(out, sum.x);
      if (n + 1 < a.n) store_out(out + 1, sum.y);
      if (n + 2 < a.n) store_out(out + 2, sum.z);
      if (n + 3 < a.n) store_out(out + 3, sum.w);
    }
    cluster_sync();  // no CTA leaves while another reads its sums
  }
}

}  // namespace ops
}  // namespace lplb

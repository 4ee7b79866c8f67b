// A whole SwiGLU mixture-of-experts layer for up to 64 tokens, in two kernels.
//
//   act[e, t, i] = silu(x[t] . gate_e[i]) * (x[t] . up_e[i])           for tokens t that chose expert e
//   out[t, h]    = sum over t's experts of weight[t, e] * (act[e, t] . down_e[h])
//
// Bound by reading the weights of the experts that were chosen, once.  So one kernel streams both
// matrices through a ring in shared memory and never stops loading: its k blocks are dealt out to the
// CTAs in equal contiguous shares (first those of gate and up, then those of down), and while the
// CTAs join their shares of `act`, the down projection's first weights already arrive.
//
// All tokens go through every chosen expert: 128 weight rows are the tensor core's M side, the tokens its N
// side, and columns of tokens that did not choose the expert are left out where results are read.
// With 64 tokens that keeps the tensor cores a fifth of the time the weights take to arrive, and
// it saves gathering rows.
//
// A share that ends inside a tile leaves a partial sum in 32 bits.  For `act` the CTA that finishes a tile
// adds its partial sums up; for `out` all CTAs share the additions.  Both go by position, not by who came
// first: the same inputs give the same bits.
//
// Shares are taken from one counter in order: a CTA that waits for `act` (or for partial sums) waits for
// shares that running CTAs hold, so the kernel ends whatever number of its CTAs is resident.
//
// Roles (384 threads): warp 0 weights (TMA), warp 1 matrix instructions, warp 2 the tokens' operand
// (TMA), warp 3 scales (8-bit weights), warps 4-11 epilogue.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>

#include "common.cuh"
#include "fp8.cuh"
#include "matmul_fp8.cuh"
#include "ops_api.h"
#include "tcgen05.cuh"

namespace lplb {
namespace ops {

constexpr int kFewTileRows = 256;  // weight rows per tile: 128 gate rows and their 128 up rows, or 256 rows of down
constexpr uint32_t kFewWeightStage = kFewTileRows * kKBytes;
constexpr int kFewMoeThreads = 384;
constexpr int kFewEpilogue = 256;
constexpr int kFewTickets = 4;
constexpr int kFewScaleSlots = 4;
constexpr uint32_t kFewScaleSlot = 3 * kScaleAtom;
constexpr int kLeastBlocks = 4;  // k blocks of a share, at least

struct FewMoeArgs {
  MoeFewPlan plan;
  const uint8_t* x_scale;    // [tokens, x_scale_ld]
  const uint8_t* w13_scale;  // [experts, 2 * inter / 128, hidden / 128]
  const uint8_t* w2_scale;   // [experts, hidden / 128, inter / 128]
  int64_t x_scale_ld;
  void* act;                 // [slots * cols, inter]
  uint8_t* act_scale;        // [slots * cols, inter / 128]
  float* partial;            // [shares, 2, 2, cols, 128] for act, then the same for out
  __nv_bfloat16* out;        // [tokens, hidden]
  int* error;
  int tokens, hidden, inter;
  int kb1, kb2;              // k blocks of 128 bytes: hidden, inter
  int shares;                // per phase, at least the tiles of the second
  int x_words, w_words;      // rows of x_scale, of the weights' scales start on 4-byte boundaries
};

// Equal contiguous shares of `total` granules.
struct Shares {
  int64_t total;  // k blocks
  int n, granule;
  // `fewest`: at least that many shares; a share then touches two tiles of total / fewest blocks at most
  __device__ __forceinline__ Shares(int64_t tiles, int kb, int shares, bool whole_tiles, int fewest) : total(tiles * kb) {
    // Whole tiles where that costs a share no more than the partial sums would.
    const int64_t even = (total + shares - 1) / shares, whole = (tiles + shares - 1) / shares * kb;
    granule = whole_tiles && whole <= even + 8 ? kb : 1;
    const int64_t most = granule == 1 ? (total + kLeastBlocks - 1) / kLeastBlocks : tiles;
    n = (int)(most < shares ? (most > fewest ? most : fewest) : shares);
  }
  __device__ __forceinline__ int64_t begin(int c) const { return c >= n ? total : total / granule * c / n * granule; }
  // the share that holds block b < total
  __device__ __forceinline__ int holder(int64_t b) const {
    int c = (int)(b * n / total);
    while (begin(c) > b) --c;
    while (begin(c + 1) <= b) ++c;
    return c;
  }
};

__device__ __forceinline__ void few_sync() { asm volatile("barrier.cta.sync.aligned 1, 256;" ::: "memory"); }
__device__ __forceinline__ void few_half_sync(int half) { asm volatile("barrier.cta.sync.aligned %0, 128;" ::"r"(2 + half) : "memory"); }
// few_sync that also says whether every thread passed true
__device__ __forceinline__ bool few_all(bool ok) {
  uint32_t all;
  __syncwarp();
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "barrier.cta.red.and.pred.aligned p, 1, 256, q;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(all)
      : "r"((uint32_t)ok)
      : "memory");
  return all != 0;
}

template <int N>
struct FewMoeLayout {
  static constexpr uint32_t kStage = kFewWeightStage + N * kKBytes;
  static constexpr int kStages = 217 * 1024 / kStage < 6 ? 217 * 1024 / kStage : 6;
  static constexpr uint32_t kScales = kStage * kStages;
  static constexpr uint32_t kMax = kScales + kFewScaleSlots * kFewScaleSlot;   // [N][4] largest magnitudes
  static constexpr uint32_t kBars = kMax + N * 16;
  static constexpr uint32_t kTotal = kBars + 8 * (2 * kStages + 2 * kFewScaleSlots + 4 + 2 * kFewTickets);
  static constexpr uint32_t kTmem = N == 16 ? 128 : N == 32 ? 256 : 512;  // 2 buffers of 2 x N columns, 12 of scales
};

__device__ __forceinline__ float few_silu(float x) { return x / (1.f + __expf(-x)); }

__device__ __forceinline__ void tmem_ld_8(uint32_t taddr, float* v) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
               : "r"(taddr)
               : "memory");
}

// Waits until *counter has reached `target`; false when the budget ran out or a role gave up.
__device__ __forceinline__ bool few_wait(const int* counter, int target, volatile int* abort) {
  if ((int)ld_acquire_gpu(reinterpret_cast<const uint32_t*>(counter)) >= target) return true;
  const uint64_t t0 = global_timer_ns();
  for (;;) {
    for (int i = 0; i < 64; ++i)
      if ((int)ld_acquire_gpu(reinterpret_cast<const uint32_t*>(counter)) >= target) return true;
    if (*abort) return false;
    if (global_timer_ns() - t0 > kWaitBudgetNs) {
      *abort = 1;
      return false;
    }
  }
}

template <bool FP8, int N>
__global__ void __launch_bounds__(kFewMoeThreads, 1)
moe_few_kernel(const __grid_constant__ CUtensorMap map_w13, const __grid_constant__ CUtensorMap map_w2, const __grid_constant__ CUtensorMap map_x,
               const __grid_constant__ CUtensorMap map_act, const FewMoeArgs a) {
  using namespace sm100;
  using L = FewMoeLayout<N>;
  constexpr int kPer = FP8 ? 128 : 64;  // values per k block
  constexpr int HN = N / 2;             // tokens per epilogue thread
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const uint32_t base = smem_u32(smem), bars = base + L::kBars;
  const uint32_t bar_full = bars, bar_empty = bars + 8 * L::kStages;
  const uint32_t bar_sfull = bar_empty + 8 * L::kStages, bar_sempty = bar_sfull + 8 * kFewScaleSlots;
  const uint32_t bar_tfull = bar_sempty + 8 * kFewScaleSlots, bar_tempty = bar_tfull + 16;
  const uint32_t bar_ticket = bar_tempty + 16, bar_ticket_read = bar_ticket + 8 * kFewTickets;
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag, s_last;
  __shared__ int s_ticket[kFewTickets];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort = &abort_flag;
  allow_successor();
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < L::kStages; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    for (int s = 0; s < kFewScaleSlots; ++s) {
      mbar_init(bar_sfull + 8 * s, 1);
      mbar_init(bar_sempty + 8 * s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar_tfull + 8 * b, 1);
      mbar_init(bar_tempty + 8 * b, kFewEpilogue / 32);
    }
    for (int s = 0; s < kFewTickets; ++s) {
      mbar_init(bar_ticket + 8 * s, 1);
      mbar_init(bar_ticket_read + 8 * s, kFewEpilogue / 32 + 2 + (FP8 ? 1 : 0));
    }
    fence_barrier_init();
    tma_prefetch_desc(&map_w13);
    tma_prefetch_desc(&map_w2);
    tma_prefetch_desc(&map_x);
    tma_prefetch_desc(&map_act);
  }
  if (warp == 1) tmem_alloc_single(smem_u32(&tmem_slot), L::kTmem);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = tmem_slot;
  wait_predecessors();

  const int slots = *a.plan.slots;                             // experts that some token chose
  const int fb = a.inter / 128, ht = a.hidden / kFewTileRows;  // tiles per expert in the first phase, tiles in the second
  const Shares one((int64_t)slots * fb, a.kb1, a.shares, true, 1), two((int64_t)ht * slots, a.kb2, a.shares, false, ht);
  const int last_ticket = 3 * a.shares;
  // The i-th ticket of this CTA, for the roles that follow the producer.
  auto ticket = [&](uint32_t i) -> int {
    const uint32_t s = i % kFewTickets;
    if (!mbar_wait(bar_ticket + 8 * s, (i / kFewTickets) & 1, abort, kWaitBudgetNs)) return last_ticket;
    return *(volatile int*)&s_ticket[s];
  };
  auto ticket_read = [&](uint32_t i) { mbar_arrive(bar_ticket_read + 8 * (i % kFewTickets)); };
  // Calls f(unit, first k block, k blocks) for every tile (first phase) or tile and slot (second) that share c touches,
  // until it returns false.
  auto walk = [&](const Shares& sh, int kb, int c, auto f) -> bool {
    const int64_t end = sh.begin(c + 1);
    for (int64_t b = sh.begin(c); b < end;) {
      const int unit = (int)(b / kb), k0 = (int)(b - (int64_t)unit * kb);
      const int n = (int)min((int64_t)(kb - k0), end - b);
      if (!f(unit, k0, n)) return false;
      b += n;
    }
    return true;
  };
  // first row of a unit's tile in w13 or w2
  auto weight_row = [&](bool first, int unit) -> int {
    if (first) return a.plan.expert[unit / fb] * 2 * a.inter + unit % fb * kFewTileRows;
    return a.plan.expert[unit % slots] * a.hidden + unit / slots * kFewTileRows;
  };

  if (warp == 0) {
    // ---------------- weights ----------------
    if (elect_one()) {
      uint32_t s = 0, ph = 0;
      for (uint32_t i = 0;; ++i) {
        const int t = min(atomicAdd(a.plan.ticket, 1), last_ticket);
        const uint32_t ts = i % kFewTickets;
        if (!mbar_wait(bar_ticket_read + 8 * ts, ((i / kFewTickets) & 1) ^ 1, abort, kWaitBudgetNs)) break;
        s_ticket[ts] = t;
        mbar_arrive(bar_ticket + 8 * ts);
        if (t >= last_ticket) break;
        if (t >= 2 * a.shares) continue;
        const bool first = t < a.shares;
        const bool ok = walk(first ? one : two, first ? a.kb1 : a.kb2, first ? t : t - a.shares, [&](int unit, int k0, int n) {
          const int row = weight_row(first, unit);
          for (int kb = k0; kb < k0 + n; ++kb) {
            if (!mbar_wait(bar_empty + 8 * s, ph ^ 1, abort, kWaitBudgetNs)) return false;
            mbar_expect_tx(bar_full + 8 * s, L::kStage);
            tma_load_2d(base + s * L::kStage, first ? &map_w13 : &map_w2, bar_full + 8 * s, kb * kPer, row);
            if (++s == L::kStages) s = 0, ph ^= 1;
          }
          return true;
        });
        if (!ok) break;
      }
    }
  } else if (warp == 1) {
    // ---------------- matrix instructions ----------------
    if (elect_one()) {
      const uint32_t idesc = FP8 ? umma_idesc_mxf8(128, N) : umma_idesc_bf16(128, N);
      const uint32_t tmem_s = tmem + 4 * N;
      uint32_t s = 0, ph = 0, ss = 0, sph = 0, seg = 0;
      for (uint32_t i = 0;; ++i) {
        const int t = ticket(i);
        ticket_read(i);
        if (t >= last_ticket) break;
        if (t >= 2 * a.shares) continue;
        const bool first = t < a.shares;
        const bool ok = walk(first ? one : two, first ? a.kb1 : a.kb2, first ? t : t - a.shares, [&](int, int k0, int n) {
          const uint32_t acc = seg & 1, acc_ph = (seg >> 1) & 1;
          ++seg;
          if (!mbar_wait(bar_tempty + 8 * acc, acc_ph ^ 1, abort, kWaitBudgetNs)) return false;
          tc_fence_after_sync();
          const uint32_t d = tmem + acc * 2 * N;
          for (int kb = k0; kb < k0 + n; ++kb) {
            if (FP8 && (kb == k0 || (kb & 3) == 0)) {
              if (!mbar_wait(bar_sfull + 8 * ss, sph, abort, kWaitBudgetNs)) return false;
              tc_fence_after_sync();
              for (int j = 0; j < 3; ++j) tmem_cp_scales(tmem_s + 4 * j, base + L::kScales + ss * kFewScaleSlot + j * kScaleAtom);
              umma_commit(bar_sempty + 8 * ss);
              if (++ss == kFewScaleSlots) ss = 0, sph ^= 1;
            }
            if (!mbar_wait(bar_full + 8 * s, ph, abort, kWaitBudgetNs)) return false;
            tc_fence_after_sync();
            const uint32_t src = base + s * L::kStage;
            const uint64_t d0 = umma_desc_sw128(src), d1 = umma_desc_sw128(src + kFewWeightStage / 2), dt = umma_desc_sw128(src + kFewWeightStage);
            const uint32_t id = FP8 ? umma_idesc_scale_byte(idesc, kb & 3) : idesc;
#pragma unroll
            for (int k = 0; k < 4; ++k) {  // 32 bytes along k inside the swizzled row
              const uint32_t more = kb != k0 || k != 0;
              if constexpr (FP8) {
                umma_mxf8(d, d0 + 2 * k, dt + 2 * k, id, tmem_s, tmem_s + 8, more);
                umma_mxf8(d + N, d1 + 2 * k, dt + 2 * k, id, tmem_s + 4, tmem_s + 8, more);
              } else {
                umma_bf16(d, d0 + 2 * k, dt + 2 * k, id, more);
                umma_bf16(d + N, d1 + 2 * k, dt + 2 * k, id, more);
              }
            }
            umma_commit(bar_empty + 8 * s);
            if (++s == L::kStages) s = 0, ph ^= 1;
          }
          umma_commit(bar_tfull + 8 * acc);
          return true;
        });
        if (!ok) break;
      }
    }
  } else if (warp == 2) {
    // ---------------- the tokens' operand ----------------
    if (elect_one()) {
      uint32_t s = 0, ph = 0;
      int ready = -1;
      for (uint32_t i = 0;; ++i) {
        const int t = ticket(i);
        ticket_read(i);
        if (t >= last_ticket) break;
        if (t >= 2 * a.shares) continue;
        const bool first = t < a.shares;
        const bool ok = walk(first ? one : two, first ? a.kb1 : a.kb2, first ? t : t - a.shares, [&](int unit, int k0, int n) {
          const int slot = first ? 0 : unit % slots;
          if (!first && slot != ready) {
            if (!few_wait(a.plan.ready + slot, fb, abort)) return false;
            fence_proxy_async_global();  // `act` was written by ordinary stores, seen through the counter
            ready = slot;
          }
          for (int kb = k0; kb < k0 + n; ++kb) {
            if (!mbar_wait(bar_empty + 8 * s, ph ^ 1, abort, kWaitBudgetNs)) return false;
            tma_load_2d(base + s * L::kStage + kFewWeightStage, first ? &map_x : &map_act, bar_full + 8 * s, kb * kPer, slot * N);
            if (++s == L::kStages) s = 0, ph ^= 1;
          }
          return true;
        });
        if (!ok) break;
      }
    }
  } else if (warp == 3) {
    // ---------------- scales ----------------
    if constexpr (FP8) {
      uint32_t ss = 0, sph = 0;
      int ready = -1;
      for (uint32_t i = 0;; ++i) {
        const int t = ticket(i);
        __syncwarp();
        if (lane == 0) ticket_read(i);
        if (!__all_sync(0xffffffffu, t < last_ticket)) break;
        if (t >= 2 * a.shares) continue;
        const bool first = t < a.shares;
        const int kbs = first ? a.kb1 : a.kb2;
        const bool ok = walk(first ? one : two, kbs, first ? t : t - a.shares, [&](int unit, int k0, int n) {
          const int slot = first ? 0 : unit % slots;
          bool go = true;
          if (!first && slot != ready) {
            go = few_wait(a.plan.ready + slot, fb, abort);
            ready = slot;
          }
          const uint8_t* w = (first ? a.w13_scale : a.w2_scale) + (int64_t)(weight_row(first, unit) / 128) * kbs;
          const uint8_t* tok = first ? a.x_scale : a.act_scale + (int64_t)slot * N * kbs;
          const int64_t ld = first ? a.x_scale_ld : kbs;
          const bool words = (kbs & 3) == 0 && a.w_words, tok_words = (kbs & 3) == 0 && (!first || a.x_words);
          for (int g = k0 / 4; 4 * g < k0 + n; ++g) {
            uint32_t tk[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const int r = lane + 32 * j;
              tk[j] = r < a.tokens && r < N && go ? scale_word(tok + r * ld, g, kbs, tok_words) : kScaleOnes;
            }
            const uint32_t w0 = scale_word(w, g, kbs, words), w1 = scale_word(w + kbs, g, kbs, words);
            go = go && mbar_wait(bar_sempty + 8 * ss, sph ^ 1, abort, kWaitBudgetNs);
            if (!__all_sync(0xffffffffu, go)) return false;
            uint8_t* dst = smem + L::kScales + ss * kFewScaleSlot + lane * 16;
            *reinterpret_cast<uint4*>(dst) = make_uint4(w0, w0, w0, w0);
            *reinterpret_cast<uint4*>(dst + kScaleAtom) = make_uint4(w1, w1, w1, w1);
            *reinterpret_cast<uint4*>(dst + 2 * kScaleAtom) = make_uint4(tk[0], tk[1], kScaleOnes, kScaleOnes);
            fence_proxy_async_shared();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_sfull + 8 * ss);
            if (++ss == kFewScaleSlots) ss = 0, sph ^= 1;
          }
          return true;
        });
        if (!ok) break;
      }
    }
  } else {
    // ---------------- epilogue ----------------
    const int half = (warp - 4) >> 2, quarter = warp & 3, et = threadIdx.x - 128;
    const int t0 = half * HN, row = quarter * 32 + lane;  // first token, row of each half tile
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const size_t part_floats = (size_t)2 * N * 128;
    float* part1 = a.partial;
    float* part2 = a.partial + (size_t)a.shares * 2 * part_floats;
    uint32_t seg = 0;
    float v0[HN], v1[HN];
    // the next accumulator into v0 and v1
    auto take = [&]() -> bool {
      const uint32_t acc = seg & 1, acc_ph = (seg >> 1) & 1;
      ++seg;
      if (!few_all(mbar_wait(bar_tfull + 8 * acc, acc_ph, abort, kWaitBudgetNs))) return false;
      tc_fence_after_sync();
      const uint32_t d = tmem + lanes + acc * 2 * N + t0;
#pragma unroll
      for (int j = 0; j < HN; j += 8) {
        tmem_ld_8(d + j, v0 + j);
        tmem_ld_8(d + N + j, v1 + j);
      }
      tmem_ld_wait();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_tempty + 8 * acc);
      return true;
    };
    for (uint32_t i = 0;; ++i) {
      const int t = ticket(i);
      __syncwarp();
      if (lane == 0) ticket_read(i);
      if (!few_all(t < last_ticket)) break;
      bool ok = true;
      if (t < a.shares) {
        // `act`: whole tiles at once, the others when their last partial sum is there
        ok = walk(one, a.kb1, t, [&](int unit, int k0, int n) {
          if (!take()) return false;
          if (n < a.kb1) {
            float* p = part1 + ((size_t)t * 2 + (k0 == 0)) * part_floats + (size_t)t0 * 128 + row;
#pragma unroll
            for (int j = 0; j < HN; ++j) {
              __stcg(p + j * 128, v0[j]);
              __stcg(p + (N + j) * 128, v1[j]);
            }
            __threadfence();
            few_sync();
            if (et == 0) s_last = atomicAdd(a.plan.tile_blocks + unit, n) + n == a.kb1;
            few_sync();
            const bool last = s_last != 0;
            if (!last) return true;
            __threadfence();
#pragma unroll
            for (int j = 0; j < HN; ++j) v0[j] = v1[j] = 0.f;
            const int64_t b0 = (int64_t)unit * a.kb1;
            for (int c = one.holder(b0); one.begin(c) < b0 + a.kb1; ++c) {
              const float* q = part1 + ((size_t)c * 2 + (one.begin(c) <= b0)) * part_floats + (size_t)t0 * 128 + row;
#pragma unroll
              for (int j = 0; j < HN; ++j) {
                v0[j] += __ldcg(q + j * 128);
                v1[j] += __ldcg(q + (N + j) * 128);
              }
            }
          }
          const int slot = unit / fb, f = unit % fb;
          const uint64_t chose = a.plan.tokens[slot] >> t0;
          if constexpr (FP8) {
            uint32_t* s_max = reinterpret_cast<uint32_t*>(smem + L::kMax);
#pragma unroll
            for (int j = 0; j < HN; ++j) {
              v0[j] = few_silu(v0[j]) * v1[j];
              const uint32_t top = __reduce_max_sync(0xffffffffu, fp8::magnitude(v0[j]));
              if (lane == 0) s_max[(t0 + j) * 4 + quarter] = top;
            }
            few_half_sync(half);
#pragma unroll
            for (int j = 0; j < HN; ++j) {
              if (!(chose >> j & 1)) continue;
              const uint4 m = *reinterpret_cast<const uint4*>(s_max + (t0 + j) * 4);
              const uint32_t e = fp8::scale_exponent(max(max(m.x, m.y), max(m.z, m.w)));
              const size_t r = (size_t)slot * N + t0 + j;
              static_cast<uint8_t*>(a.act)[r * a.inter + f * 128 + row] = (uint8_t)fp8::pack2(fp8::scaled(v0[j], fp8::reciprocal_of(e)), 0.f);
              if (row == 0) a.act_scale[r * fb + f] = (uint8_t)e;
            }
          } else {
#pragma unroll
            for (int j = 0; j < HN; ++j) {
              if (!(chose >> j & 1)) continue;
              static_cast<__nv_bfloat16*>(a.act)[((size_t)slot * N + t0 + j) * a.inter + f * 128 + row] =
                  __float2bfloat16_rn(few_silu(v0[j]) * v1[j]);  // the activations are held in the weights' type
            }
          }
          __threadfence();
          few_sync();
          if (et == 0) red_release_gpu(reinterpret_cast<uint32_t*>(a.plan.ready + slot), 1);
          return true;
        });
      } else if (t < 2 * a.shares) {
        // `out`: the share's sum over its experts, per tile
        const int c = t - a.shares;
        const int64_t end = two.begin(c + 1), tile_blocks = (int64_t)slots * a.kb2;
        float s0[HN], s1[HN];
#pragma unroll
        for (int j = 0; j < HN; ++j) s0[j] = s1[j] = 0.f;
        int64_t b = two.begin(c);
        const int first_tile = b < end ? (int)(b / tile_blocks) : 0;
        int blocks = 0;
        ok = walk(two, a.kb2, c, [&](int unit, int, int n) {
          const int slot = unit % slots, tile = unit / slots;
          const uint64_t chose = a.plan.tokens[slot] >> t0;
          const float* w = a.plan.weight + (size_t)slot * 64 + t0;
          if (!take()) return false;
#pragma unroll
          for (int j = 0; j < HN; ++j) {
            if (!(chose >> j & 1)) continue;
            const float g = __ldcg(w + j);
            s0[j] = fmaf(g, v0[j], s0[j]);
            s1[j] = fmaf(g, v1[j], s1[j]);
          }
          b += n;
          blocks += n;
          if (b == end || b == (int64_t)(tile + 1) * tile_blocks) {
            float* p = part2 + ((size_t)c * 2 + (tile != first_tile)) * part_floats + (size_t)t0 * 128 + row;
#pragma unroll
            for (int j = 0; j < HN; ++j) {
              __stcg(p + j * 128, s0[j]);
              __stcg(p + (N + j) * 128, s1[j]);
              s0[j] = s1[j] = 0.f;
            }
            __threadfence();
            few_sync();
            if (et == 0) red_release_gpu(reinterpret_cast<uint32_t*>(a.plan.out_blocks + tile), (uint32_t)blocks);
            blocks = 0;
          }
          return true;
        });
      } else {
        // sums of the shares' sums: 256 outputs of a token at a time
        const int64_t tile_blocks = (int64_t)slots * a.kb2;
        int done = -1;
        for (int u = t - 2 * a.shares; u < ht * a.tokens; u += a.shares) {
          const int tile = u / a.tokens, tok = u % a.tokens;
          if (tile != done) {
            bool there = true;
            if (et == 0) there = few_wait(a.plan.out_blocks + tile, (int)tile_blocks, abort);
            if (!few_all(there)) {
              ok = false;
              break;
            }
            __threadfence();
            done = tile;
          }
          float sum = 0.f;
          const int64_t b0 = tile * tile_blocks, b1 = b0 + tile_blocks;
          if (b1 > b0) {
            const int c1 = two.holder(b1 - 1);
            for (int c = two.holder(b0); c <= c1; ++c) {
              const int which = (int)(two.begin(c) / tile_blocks) != tile;
              sum += __ldcg(part2 + ((size_t)c * 2 + which) * part_floats + ((size_t)(et >> 7) * N + tok) * 128 + (et & 127));
            }
          }
          a.out[(size_t)tok * a.hidden + tile * kFewTileRows + et] = __float2bfloat16_rn(sum);
        }
      }
      if (!ok) break;
    }
  }
  __syncthreads();
  if (*abort) {  // a role gave up: copies in flight land before shared memory and tensor memory are released
    const uint64_t t0 = timer_ns();
    while (timer_ns() - t0 < 200000) __nanosleep(1000);
    if (threadIdx.x == 0) atomicCAS(a.error, 0, kOpsTimeout);
  }
  __syncthreads();
  if (warp == 1) tmem_dealloc_single(tmem, L::kTmem);
}

// ---- the plan -----------------------------------------------------------------------------
struct FewPlanArgs {
  MoeFewPlan plan;
  const void* idx;      // [tokens, topk]
  const float* weight;  // [tokens, topk]
  int is64, tokens, topk, experts;
  int counters;         // words from plan.ready on that start at zero
  // rows to convert to 8 bits (CTAs 1 to tokens), or null
  const __nv_bfloat16* x;
  int64_t x_ld;
  uint8_t* q;
  uint8_t* scale;
  int hidden;
};
constexpr int kFewPlanThreads = 256;

// CTA 0: which experts were chosen (slots in the experts' order), by which tokens, with which weight;
// the counters of the next kernel start at zero.  Ids outside [0, experts) choose nothing; an
// expert that a token chose more than once gets the sum of its weights, in the order of the choices.
__global__ void __launch_bounds__(kFewPlanThreads) moe_few_plan_kernel(const FewPlanArgs a) {
  allow_successor();
  wait_predecessors();
  if (blockIdx.x > 0) {
    const int64_t row = blockIdx.x - 1;
    const __nv_bfloat16* x = a.x + row * a.x_ld;
    const bool vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0;
    for (int c = threadIdx.x * 8; c < a.hidden; c += kFewPlanThreads * 8) {  // whole warps: hidden is a multiple of 256
      float v[8];
      fp8::load8(x + c, vec, 8, v);
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) top = max(top, fp8::magnitude(v[i]));
      const uint32_t e = fp8::scale_exponent(fp8::block_max(top));
      fp8::store8_e4m3(a.q + row * a.hidden + c, true, 8, fp8::pack8(v, fp8::reciprocal_of(e)));
      if ((threadIdx.x & 15) == 0) a.scale[row * (a.hidden / 128) + c / 128] = (uint8_t)e;
    }
    return;
  }
  __shared__ int s_idx[kMoeFewMaxTokens * kMoeFewMaxTopk];
  __shared__ int s_slot[kMoeFewMaxExperts];
  __shared__ uint32_t s_tokens[kMoeFewMaxExperts][2];
  const int tid = threadIdx.x, pairs = a.tokens * a.topk;
  for (int e = tid; e < a.experts; e += kFewPlanThreads) s_slot[e] = 0, s_tokens[e][0] = s_tokens[e][1] = 0;
  for (int i = tid; i < a.counters; i += kFewPlanThreads) a.plan.ready[i] = 0;
  if (tid == 0) *a.plan.ticket = 0;
  __syncthreads();
  for (int i = tid; i < pairs; i += kFewPlanThreads) {
    const int64_t e = a.is64 ? static_cast<const int64_t*>(a.idx)[i] : (int64_t)static_cast<const int*>(a.idx)[i];
    const bool ok = e >= 0 && e < a.experts;
    s_idx[i] = ok ? (int)e : -1;
    if (ok) {
      const int t = i / a.topk;
      s_slot[e] = 1;
      atomicOr(&s_tokens[e][t >> 5], 1u << (t & 31));
    }
  }
  __syncthreads();
  if (tid < 32) {
    int carry = 0;
    for (int e0 = 0; e0 < a.experts; e0 += 32) {
      const int e = e0 + tid;
      const bool on = e < a.experts && s_slot[e] != 0;
      const uint32_t ballot = __ballot_sync(0xffffffffu, on);
      const int slot = carry + __popc(ballot & ((1u << tid) - 1));
      if (on) {
        s_slot[e] = slot;
        a.plan.expert[slot] = e;
        a.plan.tokens[slot] = (uint64_t)s_tokens[e][1] << 32 | s_tokens[e][0];
      }
      carry += __popc(ballot);
    }
    if (tid == 0) *a.plan.slots = carry;
  }
  __syncthreads();
  for (int i = tid; i < pairs; i += kFewPlanThreads) {
    const int e = s_idx[i], t = i / a.topk;
    if (e < 0) continue;
    bool before = false;
    for (int j = t * a.topk; j < i; ++j) before |= s_idx[j] == e;
    if (before) continue;
    float w = a.weight[i];
    for (int j = i + 1; j < (t + 1) * a.topk; ++j)
      if (s_idx[j] == e) w += a.weight[j];
    a.plan.weight[(size_t)s_slot[e] * 64 + t] = w;
  }
}

}  // namespace ops
}  // namespace lplb

// A whole SwiGLU mixture-of-experts layer for up to 64 tokens, in two kernels.
//
//   act[e, t, i] = silu(x[t] . gate_e[i]) * (x[t] . up_e[i])           for tokens t that chose expert e
//   out[t, h]    = sum over t's experts of weight[t, e] * (act[e, t] . down_e[h])
//
// Bound by reading the weights of the experts that were chosen, once.  So one kernel streams both
// matrices through a ring in shared memory and never stops loading.  Its tasks are tiles of gate and up, expert by
// expert, then tiles of down in the same order, taken from one counter: when the last tiles of `act` are
// being made, free CTAs already work on down for the first experts, and the join of the two halves costs no time.
// (With equal contiguous shares and all of `act` awaited, 39 experts of 7168 x 2048 in 8 bits, 1.72 GB, took 332 us; now
// 272 us, the weights at 6.4 TB/s inside the kernel.)
//
// 128 weight rows are the tensor core's M side, the rows of an expert (tokens that chose it, gathered by TMA) its
// N side, rounded up to 16.  Loading all tokens for every expert instead costs no DRAM traffic, but 64 tokens
// are 8 KB more per 32 KB of weights to bring from L2, and four times the columns to multiply.
//
// Where the tiles are few, tasks are parts of a tile along k.  Their sums in 32 bits are added up by the CTA that
// finishes the tile.  Products with down stay in 32 bits per row, and all CTAs share the sums over a token's
// experts.  Both go by position, not by who came first: the same inputs give the same bits.
//
// A CTA that waits for `act` (or for products) waits for tasks with smaller numbers, which running CTAs hold and which
// wait for smaller ones at most: the kernel ends whatever number of its CTAs is resident.
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
constexpr int kFewAhead = 8;         // blocks before the end of a task that a CTA takes its next one
constexpr int kFewChunks = 4;        // chunks of scales under way
constexpr uint32_t kFewChunkBytes = (kMoeFewMaxTokens + 2) * kScaleChunk;
constexpr int kFewMaxParts = 4;      // parts of a tile along k, at most
constexpr int kFewPieces = 2;        // pieces of a product with down, at most
constexpr int kFewCols = 64;         // columns of an accumulator

// Shared memory from a 1024-byte boundary on.  The ring has as many stages as fit the largest expert's rows.
constexpr uint32_t kFewRing = 206 * 1024;
constexpr int kFewMaxStages = 6;
constexpr uint32_t kFewScalesAt = kFewRing;
constexpr uint32_t kFewChunksAt = kFewScalesAt + kFewScaleSlots * kFewScaleSlot;
constexpr uint32_t kFewMaxAt = kFewChunksAt + kFewChunks * kFewChunkBytes;  // [2 halves][2][8 tokens][4 warps] largest magnitudes
constexpr uint32_t kFewSlotsAt = kFewMaxAt + 2 * 2 * 8 * 4 * 4;
constexpr uint32_t kFewTokensAt = kFewSlotsAt + kMoeFewMaxExperts * 8;  // tokens of the rows, four more
constexpr uint32_t kFewBarsAt = kFewTokensAt + kMoeFewMaxTokens * kMoeFewMaxTopk + 16;
constexpr uint32_t kFewMoeSmem = kFewBarsAt + 8 * (2 * kFewMaxStages + 2 * kFewScaleSlots + 4 + 2 * kFewTickets) + 1024;
constexpr uint32_t kFewScaleColumns = 4 * kFewCols;  // two buffers of two accumulators, then the scales

struct FewMoeArgs {
  MoeFewPlan plan;
  const uint8_t* x_scale;    // [tokens, x_scale_ld]
  const uint8_t* w13_scale;  // [experts, 2 * inter / 128, hidden / 128]
  const uint8_t* w2_scale;   // [experts, hidden / 128, inter / 128]
  int64_t x_scale_ld;
  void* act;                 // [rows, inter]
  uint8_t* act_scale;        // [rows, inter / 128]
  float* partial;            // [tile, part][2, cols, 128]
  float* product;            // [kFewPieces, tokens * topk, hidden]
  __nv_bfloat16* out;        // [tokens, hidden]
  int* error;
  unsigned long long budget_ns;
  int tokens, topk, hidden, inter;
  int cols;                  // tokens rounded up to 16
  int kb1, kb2;              // k blocks of 128 bytes: hidden, inter
  int ctas;                  // of the second kernel
  int slots;                 // at most
  int x_words, w_words;      // rows of x_scale, of the weights' scales start on 4-byte boundaries
};

// The tasks: `parts` of every tile of `act`, then the units (slot by slot, tiles of down) whole up to `split`, in two
// pieces from there on, so that the CTAs end together.
// Division by a number that stays the same, for n * d < 2^32 (a task is looked up by five roles; five divisions of
// 20 instructions each were 1.5 us of a small layer's 22).
struct FewDivisor {
  uint32_t d, m;
  __device__ __forceinline__ explicit FewDivisor(int d_) : d((uint32_t)d_), m(d_ > 1 ? 0xFFFFFFFFu / (uint32_t)d_ + 1 : 0) {}
  __device__ __forceinline__ int of(int n) const { return d > 1 ? (int)__umulhi((uint32_t)n, m) : n; }
};
struct FewTask {
  bool first;
  int unit, slot, part, k0, k1;
};
__device__ __forceinline__ int few_parts(int tiles, int kb1, int ctas) {
  // parts (of at least eight blocks) only where the tiles leave half of the CTAs without one: adding them up costs
  // 8 us between the last block and the first product (128 tiles on 148 CTAs: 78 us, in three parts 82)
  return max(1, min(min(kFewMaxParts, kb1 / 8), tiles > 0 ? ctas / tiles : 1));
}
struct FewTasks {
  int kb1, kb2, parts, pieces, split, n1, n;
  FewDivisor by_parts, by_fb, by_ht;
  // tiles of `act` per slot, tiles of down
  __device__ __forceinline__ FewTasks(int slots, int fb, int kb1_, int ht, int kb2_, int ctas)
      : kb1(kb1_), kb2(kb2_), parts(few_parts(slots * fb, kb1_, ctas)), by_parts(parts), by_fb(fb), by_ht(ht) {
    const int units = slots * ht;
    pieces = kb2 >= 8 ? kFewPieces : 1;
    split = max(0, units - ctas);
    n1 = slots * fb * parts;
    n = n1 + split + (units - split) * pieces;
  }
  __device__ __forceinline__ FewTask at(int t) const {
    FewTask k;
    k.first = t < n1;
    if (k.first) {
      k.unit = by_parts.of(t);
      k.part = t - k.unit * parts;
      k.slot = by_fb.of(k.unit);
      k.k0 = by_parts.of(kb1 * k.part);
      k.k1 = by_parts.of(kb1 * (k.part + 1));
      return k;
    }
    t -= n1;
    k.part = 0;
    k.unit = t;
    k.k0 = 0;
    k.k1 = kb2;
    if (t >= split && pieces == 2) {
      t -= split;
      k.unit = split + (t >> 1);
      k.part = t & 1;
      if (k.part) k.k0 = kb2 / 2;
      else k.k1 = kb2 / 2;
    }
    k.slot = by_ht.of(k.unit);
    return k;
  }
};

__device__ __forceinline__ void few_sync() { asm volatile("barrier.cta.sync.aligned 1, 256;" ::: "memory"); }
__device__ __forceinline__ void few_half_sync(int half) {
  if (half == 0)
    asm volatile("barrier.cta.sync.aligned 2, 128;" ::: "memory");
  else
    asm volatile("barrier.cta.sync.aligned 3, 128;" ::: "memory");
}
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

// (__expf is documented to be off by 2 + 1.173 |x| units in the last place at most, 2^-20 of the value at 4 and 2^-17 at 30: far below
// the rounding to bf16 or 8 bits behind it)
__device__ __forceinline__ float few_silu(float x) { return x / (1.f + __expf(-x)); }

__device__ __forceinline__ void tmem_ld_8(uint32_t taddr, float (&v)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
               : "r"(taddr)
               : "memory");
}

// Waits until *counter has reached `target`; false when the budget ran out or a role gave up.
__device__ __forceinline__ bool few_wait(const int* counter, int target, volatile int* abort, uint64_t budget_ns) {
  if ((int)ld_acquire_gpu(reinterpret_cast<const uint32_t*>(counter)) >= target) return true;
  const uint64_t t0 = global_timer_ns();
  for (;;) {
    for (int i = 0; i < 64; ++i)
      if ((int)ld_acquire_gpu(reinterpret_cast<const uint32_t*>(counter)) >= target) return true;
    if (*abort) return false;
    if (global_timer_ns() - t0 > budget_ns) {
      *abort = 1;
      return false;
    }
  }
}

template <bool FP8>
__global__ void __launch_bounds__(kFewMoeThreads, 1)
moe_few_kernel(const __grid_constant__ CUtensorMap map_w13, const __grid_constant__ CUtensorMap map_w2, const __grid_constant__ CUtensorMap map_x,
               const __grid_constant__ CUtensorMap map_act, const FewMoeArgs a) {
  using namespace sm100;
  constexpr int kPer = FP8 ? 128 : 64;  // values per k block
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const uint32_t base = smem_u32(smem), bars = base + kFewBarsAt;
  const uint32_t bar_full = bars, bar_empty = bars + 8 * kFewMaxStages;
  const uint32_t bar_sfull = bar_empty + 8 * kFewMaxStages, bar_sempty = bar_sfull + 8 * kFewScaleSlots;
  const uint32_t bar_tfull = bar_sempty + 8 * kFewScaleSlots, bar_tempty = bar_tfull + 16;
  const uint32_t bar_ticket = bar_tempty + 16, bar_ticket_read = bar_ticket + 8 * kFewTickets;
  int2* s_slot = reinterpret_cast<int2*>(smem + kFewSlotsAt);
  uint8_t* s_token = smem + kFewTokensAt;
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag, s_last, s_most;
  __shared__ int s_ticket[kFewTickets];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort = &abort_flag;
  allow_successor();
  if (threadIdx.x == 0) {
    abort_flag = 0;
    s_most = 0;
    for (int s = 0; s < kFewMaxStages; ++s) {
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
  if (warp == 1) tmem_alloc_single(smem_u32(&tmem_slot), 512);
  __syncthreads();
  wait_predecessors();
  // all that the plan holds in one round trip, the first ticket too
  int first_ticket = 0;
  if (threadIdx.x == 0) first_ticket = atomicAdd(a.plan.ticket, 1);
  const int slots = *a.plan.slots;
  for (int i = threadIdx.x; i < a.slots; i += kFewMoeThreads) {
    const int2 s = a.plan.slot[i];
    if (i >= slots) break;
    s_slot[i] = s;
    atomicMax(&s_most, s.y & 255);
  }
  for (int i = threadIdx.x; i < a.tokens * a.topk + 4; i += kFewMoeThreads) s_token[i] = a.plan.token[i];
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = tmem_slot;
  const uint32_t stage_bytes = kFewWeightStage + (uint32_t)(s_most + 15) / 16 * 16 * kKBytes;
  const uint32_t stages = min((uint32_t)kFewMaxStages, kFewRing / stage_bytes);
  const int fb = a.inter / 128, ht = a.hidden / kFewTileRows;  // tiles per expert in the first phase, tiles in the second
  const FewTasks tasks(slots, fb, a.kb1, ht, a.kb2, a.ctas);
  const int last_ticket = tasks.n;
  // The i-th ticket of this CTA, for the roles that follow the producer.
  auto ticket = [&](uint32_t i) -> int {
    const uint32_t s = i % kFewTickets;
    if (!mbar_wait(bar_ticket + 8 * s, (i / kFewTickets) & 1, abort, a.budget_ns)) return last_ticket;
    return *(volatile int*)&s_ticket[s];
  };
  auto ticket_read = [&](uint32_t i) { mbar_arrive(bar_ticket_read + 8 * (i % kFewTickets)); };
  // first row of a task's tile in w13 or w2
  auto weight_row = [&](const FewTask& k) -> int {
    const int tile = k.unit - k.slot * (k.first ? fb : ht);
    return s_slot[k.slot].x * (k.first ? 2 * a.inter : a.hidden) + tile * kFewTileRows;
  };

  if (warp == 0) {
    // ---------------- weights ----------------
    if (lane == 0) {
      uint32_t s = 0, ph = 0;
      // The next task is taken, and announced, a few blocks before the end of this one: early enough for its scales,
      // late enough to go to the CTA that is ahead.
      auto announce = [&](uint32_t i) -> int {
        const uint32_t ts = i % kFewTickets;
        const int t = min(i == 0 ? first_ticket : atomicAdd(a.plan.ticket, 1), last_ticket);
        if (!mbar_wait(bar_ticket_read + 8 * ts, ((i / kFewTickets) & 1) ^ 1, abort, a.budget_ns)) return last_ticket;
        s_ticket[ts] = t;
        mbar_arrive(bar_ticket + 8 * ts);
        return t;
      };
      int next = announce(0);
      for (uint32_t i = 0; next < last_ticket; ++i) {
        const FewTask k = tasks.at(next);
        bool announced = false, ok = true;
        const int row = weight_row(k), rows = s_slot[k.slot].y & 255;
        const uint32_t bytes = kFewWeightStage + (k.first ? (rows + 3) / 4 * 4 : (rows + 15) / 16 * 16) * kKBytes;
        for (int kb = k.k0; kb < k.k1; ++kb) {
          if (!announced && k.k1 - kb <= kFewAhead) {
            announced = true;
            next = announce(i + 1);
          }
          ok = mbar_wait(bar_empty + 8 * s, ph ^ 1, abort, a.budget_ns);
          if (!ok) break;
          mbar_expect_tx(bar_full + 8 * s, bytes);
          tma_load_2d(base + s * stage_bytes, k.first ? &map_w13 : &map_w2, bar_full + 8 * s, kb * kPer, row);
          if (++s == stages) s = 0, ph ^= 1;
        }
        if (!ok) break;
      }
    }
  } else if (warp == 1) {
    // ---------------- matrix instructions ----------------
    if (elect_one()) {
      const uint32_t tmem_s = tmem + kFewScaleColumns;
      uint32_t s = 0, ph = 0, ss = 0, sph = 0, seg = 0;
      bool ok = true;
      for (uint32_t i = 0; ok; ++i) {
        const int t = ticket(i);
        ticket_read(i);
        if (t >= last_ticket) break;
        const FewTask task = tasks.at(t);
        const uint32_t acc = seg & 1, acc_ph = (seg >> 1) & 1;
        ++seg;
        const int cols = ((s_slot[task.slot].y & 255) + 15) / 16 * 16;
        const uint32_t idesc = FP8 ? umma_idesc_mxf8(128, cols) : umma_idesc_bf16(128, cols);
        if (!mbar_wait(bar_tempty + 8 * acc, acc_ph ^ 1, abort, a.budget_ns)) break;
        tc_fence_after_sync();
        const uint32_t d = tmem + acc * 2 * kFewCols;
        for (int kb = task.k0; kb < task.k1; ++kb) {
          if (FP8 && (kb == task.k0 || (kb & 3) == 0)) {
            ok = mbar_wait(bar_sfull + 8 * ss, sph, abort, a.budget_ns);
            if (!ok) break;
            tc_fence_after_sync();
            for (int j = 0; j < 3; ++j) tmem_cp_scales(tmem_s + 4 * j, base + kFewScalesAt + ss * kFewScaleSlot + j * kScaleAtom);
            umma_commit(bar_sempty + 8 * ss);
            if (++ss == kFewScaleSlots) ss = 0, sph ^= 1;
          }
          ok = mbar_wait(bar_full + 8 * s, ph, abort, a.budget_ns);
          if (!ok) break;
          tc_fence_after_sync();
          const uint32_t src = base + s * stage_bytes;
          const uint64_t d0 = umma_desc_sw128(src), d1 = umma_desc_sw128(src + kFewWeightStage / 2), dt = umma_desc_sw128(src + kFewWeightStage);
          const uint32_t id = FP8 ? umma_idesc_scale_byte(idesc, kb & 3) : idesc;
#pragma unroll
          for (int k = 0; k < 4; ++k) {  // 32 bytes along k inside the swizzled row
            const uint32_t more = kb != task.k0 || k != 0;
            if constexpr (FP8) {
              umma_mxf8(d, d0 + 2 * k, dt + 2 * k, id, tmem_s, tmem_s + 8, more);
              umma_mxf8(d + kFewCols, d1 + 2 * k, dt + 2 * k, id, tmem_s + 4, tmem_s + 8, more);
            } else {
              umma_bf16(d, d0 + 2 * k, dt + 2 * k, id, more);
              umma_bf16(d + kFewCols, d1 + 2 * k, dt + 2 * k, id, more);
            }
          }
          umma_commit(bar_empty + 8 * s);
          if (++s == stages) s = 0, ph ^= 1;
        }
        if (ok) umma_commit(bar_tfull + 8 * acc);
      }
    }
  } else if (warp == 2) {
    // ---------------- the rows' operand: tokens gathered from x, rows of `act` ----------------
    if (elect_one()) {
      uint32_t s = 0, ph = 0;
      int ready = -1;
      bool ok = true;
      for (uint32_t i = 0; ok; ++i) {
        const int t = ticket(i);
        ticket_read(i);
        if (t >= last_ticket) break;
        const FewTask task = tasks.at(t);
        const int slot = task.slot, row0 = s_slot[slot].y >> 8, rows = s_slot[slot].y & 255;
        if (!task.first && slot != ready) {
          if (!few_wait(a.plan.ready + slot, fb, abort, a.budget_ns)) break;
          fence_proxy_async_global();  // `act` was written by ordinary stores, seen through the counter
          ready = slot;
        }
        for (int kb = task.k0; kb < task.k1; ++kb) {
          ok = mbar_wait(bar_empty + 8 * s, ph ^ 1, abort, a.budget_ns);
          if (!ok) break;
          const uint32_t dst = base + s * stage_bytes + kFewWeightStage;
          if (task.first) {
            for (int j = 0; j < rows; j += 4) {
              const uint8_t* tok = s_token + row0 + j;  // beyond the last row: any token's
              const int y[4] = {tok[0], tok[1], tok[2], tok[3]};
              tma_gather4(dst + j * kKBytes, &map_x, bar_full + 8 * s, kb * kPer, y);
            }
          } else {
            for (int j = 0; j < rows; j += 16) tma_load_2d(dst + j * kKBytes, &map_act, bar_full + 8 * s, kb * kPer, row0 + j);
          }
          if (++s == stages) s = 0, ph ^= 1;
        }
      }
    }
  } else if (warp == 3) {
    // ---------------- scales ----------------
    if constexpr (FP8) {
      // Chunks of 16 blocks go through a ring by asynchronous copies, up to four of them under way, so that the next tile's
      // and the next share's scales are there when the matrix instructions reach them.
      uint32_t ss = 0, sph = 0, ticket_i = 0, queue = 0, put = 0, got = 0;
      int kb = 0, flight = 0, ready = -1;
      FewTask task;
      task.k1 = 0;
      bool more = true, ok = true;
      // 1: there is a chunk at block kb of `task`; 0: not known yet (`wait`: never); -1: none is left
      auto look = [&](bool wait) -> int {
        if (kb >= task.k1) {
          const uint32_t s = ticket_i % kFewTickets;
          if (!wait && !__all_sync(0xffffffffu, mbar_test(bar_ticket + 8 * s, (ticket_i / kFewTickets) & 1))) return 0;
          const int t = ticket(ticket_i);
          __syncwarp();
          if (lane == 0) ticket_read(ticket_i);
          ++ticket_i;
          if (!__all_sync(0xffffffffu, t < last_ticket)) return -1;
          task = tasks.at(t);
          kb = task.k0;
        }
        const int slot = task.slot;
        if (!task.first && slot != ready) {
          bool there;
          if (wait)
            there = few_wait(a.plan.ready + slot, fb, abort, a.budget_ns);
          else
            there = (int)ld_acquire_gpu(reinterpret_cast<const uint32_t*>(a.plan.ready + slot)) >= fb;
          if (!__all_sync(0xffffffffu, there)) return wait ? -1 : 0;
          ready = slot;
        }
        return 1;
      };
      auto fetch = [&]() {
        const bool first = task.first;
        const int kbs = first ? a.kb1 : a.kb2, k0 = kb, chunk = k0 / kScaleChunk, k1 = min(task.k1, (chunk + 1) * kScaleChunk);
        const int slot = task.slot, row0 = s_slot[slot].y >> 8, rows = s_slot[slot].y & 255;
        const bool w_words = (kbs & 3) == 0 && a.w_words, row_words = (kbs & 3) == 0 && (!first || a.x_words);
        const uint8_t* w = (first ? a.w13_scale : a.w2_scale) + (int64_t)(weight_row(task) / 128) * kbs;
        uint8_t* dst = smem + kFewChunksAt + put % kFewChunks * kFewChunkBytes;
        auto row_of = [&](int r) { return first ? a.x_scale + s_token[row0 + r] * a.x_scale_ld : a.act_scale + (int64_t)(row0 + r) * kbs; };
        auto copy = [&](uint8_t* to, const uint8_t* row, int i) {  // word i of the chunk
          const int kb = chunk * kScaleChunk + 4 * i;
          if (kb < kbs) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(to) + 4 * i), "l"(row + kb) : "memory");
        };
        if (w_words && row_words) {
          if (lane < 8) copy(dst + (kMoeFewMaxTokens + (lane >> 2)) * kScaleChunk, w + (lane >> 2) * kbs, lane & 3);
          for (int r = lane; r < rows; r += 32) {
            const uint8_t* src = row_of(r);
#pragma unroll
            for (int i = 0; i < 4; ++i) copy(dst + r * kScaleChunk, src, i);
          }
        } else {  // copies of words want words: by way of registers
          ScaleChunk<false> c[3];
          c[0].fetch(row_of(min(lane, rows - 1)), chunk, kbs);
          c[1].fetch(row_of(min(lane + 32, rows - 1)), chunk, kbs);
          c[2].fetch(w + (lane & 1) * kbs, chunk, kbs);
          uint4* to = reinterpret_cast<uint4*>(dst);
          to[lane] = make_uint4(c[0].word(0), c[0].word(1), c[0].word(2), c[0].word(3));
          to[lane + 32] = make_uint4(c[1].word(0), c[1].word(1), c[1].word(2), c[1].word(3));
          if (lane < 2) to[kMoeFewMaxTokens + lane] = make_uint4(c[2].word(0), c[2].word(1), c[2].word(2), c[2].word(3));
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        queue |= (uint32_t)((k0 & (kScaleChunk - 1)) | (k1 - k0 - 1) << 4) << (8 * flight);
        ++put;
        ++flight;
        kb = k1;
      };
      while (ok) {
        while (more && flight < kFewChunks) {
          const int there = look(flight == 0);
          if (there == 0) break;
          if (there < 0)
            more = false;
          else
            fetch();
        }
        if (flight == 0) break;
        if (flight == 1) asm volatile("cp.async.wait_group 0;" ::: "memory");
        else if (flight == 2) asm volatile("cp.async.wait_group 1;" ::: "memory");
        else if (flight == 3) asm volatile("cp.async.wait_group 2;" ::: "memory");
        else asm volatile("cp.async.wait_group 3;" ::: "memory");
        __syncwarp();
        const int k0 = queue & 15, k1 = k0 + (queue >> 4 & 15) + 1;  // of the chunk's blocks
        queue >>= 8;
        const uint8_t* src = smem + kFewChunksAt + got % kFewChunks * kFewChunkBytes;
        for (int i = k0 / 4; ok && 4 * i < k1; ++i) {
          const uint32_t* word = reinterpret_cast<const uint32_t*>(src) + i;
          const uint32_t w0 = word[kMoeFewMaxTokens * 4], w1 = word[kMoeFewMaxTokens * 4 + 4], r0 = word[lane * 4], r1 = word[(lane + 32) * 4];
          ok = __all_sync(0xffffffffu, mbar_wait(bar_sempty + 8 * ss, sph ^ 1, abort, a.budget_ns));
          if (!ok) break;
          uint8_t* dst = smem + kFewScalesAt + ss * kFewScaleSlot + lane * 16;
          *reinterpret_cast<uint4*>(dst) = make_uint4(w0, w0, w0, w0);
          *reinterpret_cast<uint4*>(dst + kScaleAtom) = make_uint4(w1, w1, w1, w1);
          *reinterpret_cast<uint4*>(dst + 2 * kScaleAtom) = make_uint4(r0, r1, kScaleOnes, kScaleOnes);
          fence_proxy_async_shared();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar_sfull + 8 * ss);
          if (++ss == kFewScaleSlots) ss = 0, sph ^= 1;
        }
        ++got;
        --flight;
      }
      asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
  } else {
    // ---------------- epilogue ----------------
    // Thread: a row of each half tile, and of the columns every second group of eight.
    const int half = (warp - 4) >> 2, quarter = warp & 3, et = threadIdx.x - 128;
    const int row = quarter * 32 + lane;
    const size_t part_floats = (size_t)2 * a.cols * 128;
    uint32_t seg = 0, turn = 0;
    float v0[8], v1[8];
    auto column = [&](int c0) {  // eight columns of both accumulators
      const uint32_t d = tmem + ((uint32_t)(quarter * 32) << 16) + (seg & 1) * 2 * kFewCols + c0;
      __syncwarp();
      tmem_ld_8(d, v0);
      tmem_ld_8(d + kFewCols, v1);
      tmem_ld_wait();
    };
    auto arrived = [&]() -> bool {
      if (!few_all(mbar_wait(bar_tfull + 8 * (seg & 1), (seg >> 1) & 1, abort, a.budget_ns))) return false;
      tc_fence_after_sync();
      return true;
    };
    auto release = [&]() {
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_tempty + 8 * (seg & 1));
      ++seg;
    };
    for (uint32_t i = 0;; ++i) {
      const int t = ticket(i);
      __syncwarp();
      if (lane == 0) ticket_read(i);
      if (!few_all(!*abort)) break;
      if (t < last_ticket) {
        const FewTask task = tasks.at(t);
        const int unit = task.unit, slot = task.slot, row0 = s_slot[slot].y >> 8, rows = s_slot[slot].y & 255;
        if (!arrived()) break;
        if (task.first) {
          // `act`: whole tiles at once, the others when the sums of all their parts are there
          const int f = unit - slot * fb;
          const bool whole = tasks.parts == 1;
          if (!whole) {
            float* p = a.partial + (size_t)t * part_floats + row;
            for (int c0 = half * 8; c0 < rows; c0 += 16) {
              column(c0);
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                if (c0 + j >= rows) break;
                __stcg(p + (c0 + j) * 128, v0[j]);
                __stcg(p + (a.cols + c0 + j) * 128, v1[j]);
              }
            }
            release();
            few_sync();
            if (et == 0) {  // one thread's fences, for all that the barriers put in front of and behind it
              __threadfence();
              s_last = atomicAdd(a.plan.tile_parts + unit, 1) == tasks.parts - 1;
              __threadfence();
            }
            few_sync();
            if (s_last == 0) continue;
          }
          for (int c0 = half * 8; c0 < rows; c0 += 16) {
            if (whole) {
              column(c0);
            } else {
              // all loads first: each takes microseconds while weights stream in
              const float* q = a.partial + (size_t)(t - task.part) * part_floats + row;
              float f[kFewMaxParts][16];
#pragma unroll
              for (int i = 0; i < kFewMaxParts; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                  f[i][j] = f[i][8 + j] = 0.f;
                  if (i < tasks.parts && c0 + j < rows) {
                    f[i][j] = __ldcg(q + i * part_floats + (c0 + j) * 128);
                    f[i][8 + j] = __ldcg(q + i * part_floats + (a.cols + c0 + j) * 128);
                  }
                }
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                v0[j] = f[0][j], v1[j] = f[0][8 + j];
#pragma unroll
                for (int i = 1; i < kFewMaxParts; ++i) v0[j] += f[i][j], v1[j] += f[i][8 + j];
              }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) v0[j] = few_silu(v0[j]) * v1[j];
            if constexpr (FP8) {
              // 128 features of a row share a scale: four warps
              uint32_t* s_max = reinterpret_cast<uint32_t*>(smem + kFewMaxAt) + (half * 2 + (turn & 1)) * 32;
              ++turn;
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const uint32_t top = __reduce_max_sync(0xffffffffu, fp8::magnitude(v0[j]));
                if (lane == 0) s_max[j * 4 + quarter] = top;
              }
              few_half_sync(half);
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                if (c0 + j >= rows) break;
                const uint4 m = *reinterpret_cast<const uint4*>(s_max + j * 4);
                const uint32_t e = fp8::scale_exponent(max(max(m.x, m.y), max(m.z, m.w)));
                const size_t r = row0 + c0 + j;
                static_cast<uint8_t*>(a.act)[r * a.inter + f * 128 + row] = (uint8_t)fp8::pack2(fp8::scaled(v0[j], fp8::reciprocal_of(e)), 0.f);
                if (row == 0) a.act_scale[r * fb + f] = (uint8_t)e;
              }
            } else {
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                if (c0 + j >= rows) break;  // the activations are held in the weights' type
                static_cast<__nv_bfloat16*>(a.act)[(size_t)(row0 + c0 + j) * a.inter + f * 128 + row] = __float2bfloat16_rn(v0[j]);
              }
            }
          }
          if (whole) release();
          few_sync();
          if (et == 0) red_release_gpu(reinterpret_cast<uint32_t*>(a.plan.ready + slot), 1);
        } else {
          // a product with down, or a piece of it
          const int tile = unit - slot * ht;
          float* p = a.product + ((size_t)task.part * a.tokens * a.topk + row0) * a.hidden + tile * kFewTileRows + row;
          for (int c0 = half * 8; c0 < rows; c0 += 16) {
            column(c0);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              if (c0 + j >= rows) break;
              __stcg(p + (size_t)(c0 + j) * a.hidden, v0[j]);
              __stcg(p + (size_t)(c0 + j) * a.hidden + 128, v1[j]);
            }
          }
          release();
          few_sync();
          if (et == 0) red_release_gpu(reinterpret_cast<uint32_t*>(a.plan.products), 1);
        }
      } else {
        // Nothing is left to take.  A token's sum over its experts, 128 outputs to a warp at a time; every CTA of the
        // grid comes by here, and all products are made or being made.
        const int parts = a.hidden / 128, step = (int)gridDim.x * 8, n_out = parts * a.tokens;
        int u = (int)blockIdx.x * 8 + warp - 4;
        auto choice = [&](int u) {  // lane k looks up choice k
          return u < n_out && lane < a.topk ? a.plan.pair[u / parts * a.topk + lane] : make_int2(-1, 0);
        };
        int2 next = choice(u);
        bool there = true;
        if (lane == 0) there = few_wait(a.plan.products, tasks.n - tasks.n1, abort, a.budget_ns);
        if (!__all_sync(0xffffffffu, there)) break;
        __threadfence();
        for (; u < n_out; u += step) {
          const int tok = u / parts, part = u - tok * parts, tile = part >> 1;
          const int2 mine = next;
          next = choice(u + step);
          const int pieces = mine.x >= 0 && (mine.x & 1023) * ht + tile >= tasks.split ? tasks.pieces : 1;
          const float4* p = reinterpret_cast<const float4*>(a.product + (size_t)part * 128) + lane;
          const size_t piece = (size_t)a.tokens * a.topk * a.hidden / 4;
          float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
          for (int k0 = 0; k0 < a.topk; k0 += 8) {
            float4 y[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const int at = __shfl_sync(0xffffffffu, mine.x, (k0 + j) & 31);
              y[j] = make_float4(0.f, 0.f, 0.f, 0.f);
              if (k0 + j < a.topk && at >= 0) y[j] = __ldcg(p + (size_t)(at >> 10) * (a.hidden / 4));
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const int at = __shfl_sync(0xffffffffu, mine.x, (k0 + j) & 31), count = __shfl_sync(0xffffffffu, pieces, (k0 + j) & 31);
              const float w = __int_as_float(__shfl_sync(0xffffffffu, mine.y, (k0 + j) & 31));
              if (k0 + j >= a.topk || at < 0) continue;
              for (int q = 1; q < count; ++q) {
                const float4 f = __ldcg(p + q * piece + (size_t)(at >> 10) * (a.hidden / 4));
                y[j].x += f.x, y[j].y += f.y, y[j].z += f.z, y[j].w += f.w;
              }
              sum.x = fmaf(w, y[j].x, sum.x), sum.y = fmaf(w, y[j].y, sum.y);
              sum.z = fmaf(w, y[j].z, sum.z), sum.w = fmaf(w, y[j].w, sum.w);
            }
          }
          __nv_bfloat162 lo = __floats2bfloat162_rn(sum.x, sum.y), hi = __floats2bfloat162_rn(sum.z, sum.w);
          uint2 packed = make_uint2(*reinterpret_cast<uint32_t*>(&lo), *reinterpret_cast<uint32_t*>(&hi));
          *reinterpret_cast<uint2*>(a.out + (size_t)tok * a.hidden + part * 128 + lane * 4) = packed;
        }
        break;
      }
    }
  }
  __syncthreads();
  if (*abort) {  // a role gave up: copies in flight land before shared memory and tensor memory are released
    const uint64_t t0 = timer_ns();
    while (timer_ns() - t0 < 200000) __nanosleep(1000);
    if (threadIdx.x == 0) atomicCAS(a.error, 0, kOpsTimeout);
  }
  __syncthreads();
  if (warp == 1) tmem_dealloc_single(tmem, 512);
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
    for (int c = threadIdx.x * 8; c < a.hidden; c += kFewPlanThreads * 8) {  // whole warps: hidden is a multiple of 256
      float2 v[4];
      fp8::unpack(fp8::load_raw<true>(x + c, 8), v);
      const uint32_t e = fp8::scale_exponent(fp8::block_max(fp8::magnitude8(v)));
      fp8::store8_e4m3<true>(a.q + row * a.hidden + c, 8, fp8::pack8(v, fp8::reciprocal_of(e), fp8::all_finite(v)));
      if ((threadIdx.x & 15) == 0) a.scale[row * (a.hidden / 128) + c / 128] = (uint8_t)e;
    }
    return;
  }
  __shared__ int s_idx[kMoeFewMaxTokens * kMoeFewMaxTopk];
  __shared__ int2 s_slot[kMoeFewMaxExperts];  // slot, first row
  __shared__ uint32_t s_tokens[kMoeFewMaxExperts][2];
  const int tid = threadIdx.x, pairs = a.tokens * a.topk;
  for (int e = tid; e < a.experts; e += kFewPlanThreads) s_tokens[e][0] = s_tokens[e][1] = 0;
  for (int i = tid; i < a.counters; i += kFewPlanThreads) a.plan.ready[i] = 0;
  for (int i = tid; i < pairs + 4; i += kFewPlanThreads) a.plan.token[i] = 0;
  if (tid == 0) *a.plan.ticket = 0;
  __syncthreads();
  for (int i = tid; i < pairs; i += kFewPlanThreads) {
    const int64_t e = a.is64 ? static_cast<const int64_t*>(a.idx)[i] : (int64_t)static_cast<const int*>(a.idx)[i];
    const bool ok = e >= 0 && e < a.experts;
    s_idx[i] = ok ? (int)e : -1;
    if (ok) {
      const int t = i / a.topk;
      atomicOr(&s_tokens[e][t >> 5], 1u << (t & 31));
    }
  }
  __syncthreads();
  if (tid < 32) {
    int slot0 = 0, row0 = 0;
    for (int e0 = 0; e0 < a.experts; e0 += 32) {
      const int e = e0 + tid;
      const int n = e < a.experts ? __popc(s_tokens[e][0]) + __popc(s_tokens[e][1]) : 0;
      const uint32_t ballot = __ballot_sync(0xffffffffu, n > 0);
      int before = n;  // rows of the experts in front
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, before, o);
        if (tid >= o) before += up;
      }
      if (n > 0) {
        const int slot = slot0 + __popc(ballot & ((1u << tid) - 1));
        s_slot[e] = make_int2(slot, row0 + before - n);
        a.plan.slot[slot] = make_int2(e, (row0 + before - n) << 8 | n);
      }
      slot0 += __popc(ballot);
      row0 += __shfl_sync(0xffffffffu, before, 31);
    }
    if (tid == 0) *a.plan.slots = slot0;
  }
  __syncthreads();
  for (int i = tid; i < pairs; i += kFewPlanThreads) {
    const int e = s_idx[i], t = i / a.topk;
    bool mine = e >= 0;  // the first of a token's choices of this expert
    for (int j = t * a.topk; j < i; ++j) mine &= s_idx[j] != e;
    int2 pair = make_int2(-1, 0);
    if (mine) {
      float w = a.weight[i];
      for (int j = i + 1; j < (t + 1) * a.topk; ++j)
        if (s_idx[j] == e) w += a.weight[j];
      const int2 s = s_slot[e];
      const uint64_t chose = (uint64_t)s_tokens[e][1] << 32 | s_tokens[e][0];
      const int r = __popcll(chose & ((1ull << t) - 1));  // the token's place among the slot's rows
      a.plan.token[s.y + r] = (uint8_t)t;
      pair = make_int2((s.y + r) << 10 | s.x, __float_as_int(w));
    }
    a.plan.pair[i] = pair;
  }
}

}  // namespace ops
}  // namespace lplb

// Rows to their experts and back by bulk copies: for rows of whole 16-byte words on 16-byte boundaries.
//
// All three kernels are bound by DRAM and hold 190 KB of rows per SM under way, in a ring of slots in shared memory; one CTA per SM goes
// through the batch.  take_rows never has a row in registers: a slot is loaded once and stored to all of its places.  combine_rows
// and its gradient load a piece of every row of a token into one slot; eight warps add it up from there.
//
// 8192 tokens x 8 rows of 7168 in bf16 (copy rate 6541 GB/s): see the launchers.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"
#include "experts_api.h"
#include "tcgen05.cuh"

namespace lplb {
namespace ops {

constexpr uint32_t kBulkRing = 190 * 1024;
constexpr int kBulkSlots = 16;          // at most
constexpr int kBulkTurns = kBulkSlots + 1;
constexpr uint32_t kBulkBars = 512;     // full and empty of every slot, and one per turn
static_assert((2 * kBulkSlots + kBulkTurns) * 8 <= kBulkBars, "barriers");
constexpr size_t kBulkSmem = 128 + kBulkRing + kBulkBars;

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}
__device__ __forceinline__ void bulk_store(void* dst, uint32_t src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
// until at most N of this thread's groups still read shared memory
template <int N>
__device__ __forceinline__ void bulk_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}

struct BulkArgs {
  int* status;
  unsigned long long budget_ns;
  int64_t pieces;      // of a row
  uint32_t piece;      // bytes, but of the last; a multiple of 16
  uint32_t slot;       // bytes of a slot
  int whole;           // combine_rows: a CTA has all pieces of a token (always in the gradient)
  int slots;
};

// ---- take_rows ------------------------------------------------------------------------------------------
// A warp; a slot holds a piece of a token's row, a lane sends it to one of the token's places.  Before a slot is loaded again its
// stores, `kTakeBehind` items back, have read it.
constexpr int kTakeBehind = 5;
constexpr uint32_t kTakeMostPiece = 16 * 1024;

static __global__ void __launch_bounds__(32) take_rows_bulk_kernel(const TakeRows t, const BulkArgs a) {
  using namespace sm100;
  extern __shared__ uint8_t bulk_shared[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(bulk_shared) + 127) & ~(uintptr_t)127);
  const uint32_t ring = smem_u32(smem), zero = ring + a.slots * a.slot, bars = ring + kBulkRing;
  __shared__ int abort_flag;
  const int lane = threadIdx.x;
  if (lane == 0) {
    abort_flag = 0;
    for (int s = 0; s < a.slots; ++s) mbar_init(bars + 8 * s, 1);
    fence_barrier_init();
  }
  for (uint32_t i = lane * 16; i < a.slot; i += 32 * 16) *reinterpret_cast<uint4*>(smem + a.slots * a.slot + i) = make_uint4(0, 0, 0, 0);
  fence_proxy_async_shared();
  __syncwarp();
  wait_predecessors();
  allow_successor();
  const int64_t items = t.tokens * a.pieces, n_rows = t.tokens * t.topk;
  const int64_t mine = (items - blockIdx.x + gridDim.x - 1) / gridDim.x;  // of this CTA: blockIdx.x, and gridDim.x apart
  const uint8_t* x = static_cast<const uint8_t*>(t.x);
  uint8_t* rows = static_cast<uint8_t*>(t.rows);
  auto locate = [&](int64_t n, int64_t& token, int64_t& from, uint32_t& bytes) {
    const int64_t item = blockIdx.x + n * gridDim.x;
    token = item / a.pieces;
    from = (item - token * a.pieces) * a.piece;
    bytes = (uint32_t)min((int64_t)a.piece, t.row_bytes - from);
  };
  auto load = [&](int64_t n) {
    int64_t token, from;
    uint32_t bytes;
    locate(n, token, from, bytes);
    const uint32_t s = (uint32_t)(n % a.slots);
    mbar_expect_tx(bars + 8 * s, bytes);
    bulk_load(ring + s * a.slot, x + token * t.ld_bytes + from, bytes, bars + 8 * s);
  };
  if (lane == 0)
    for (int64_t n = 0; n < min(mine, (int64_t)a.slots); ++n) load(n);
  volatile int* abort = &abort_flag;
  // Places are fetched for as many items as the warp has lanes for, a batch ahead: beside a busy TMA an ordinary load takes microseconds.
  const int batch = t.topk < 32 ? 32 / t.topk : 1;
  const int of = lane / t.topk, k0 = lane - of * t.topk;  // this lane's item of a batch, and its choice
  int place = -1, source = 0, next_place = -1, next_source = 0;
  auto fetch = [&](int64_t n) {
    next_place = -1, next_source = 0;
    if (n + of >= mine || of >= batch) return;
    int64_t token, from;
    uint32_t bytes;
    locate(n + of, token, from, bytes);
    next_place = t.place[token * t.topk + k0], next_source = t.source[token * t.topk + k0];
  };
  fetch(0);
  int in_batch = batch - 1;
  for (int64_t n = 0; n < mine; ++n) {
    if (++in_batch == batch) {
      in_batch = 0;
      place = next_place, source = next_source;
      fetch(n + batch);
    }
    int64_t token, from;
    uint32_t bytes;
    locate(n, token, from, bytes);
    const uint32_t s = (uint32_t)(n % a.slots);
    if (!__all_sync(0xffffffffu, mbar_wait(bars + 8 * s, (uint32_t)(n / a.slots) & 1, abort, a.budget_ns))) break;
    auto send = [&](int to, int from_pair, int k) {
      if (to >= 0 && to < n_rows) bulk_store(rows + to * t.row_bytes + from, ring + s * a.slot, bytes);
      if (from_pair < 0) bulk_store(rows + (token * t.topk + k) * t.row_bytes + from, zero, bytes);  // a row that nobody has
    };
    if (of == in_batch) send(place, source, k0);
    for (int k = lane + 32; k < t.topk; k += 32) send(t.place[token * t.topk + k], t.source[token * t.topk + k], k);
    bulk_commit();
    if (n >= kTakeBehind) {
      bulk_wait_read<kTakeBehind>();
      __syncwarp();
      if (lane == 0 && n - kTakeBehind + a.slots < mine) load(n - kTakeBehind + a.slots);
    }
  }
  bulk_wait_read<0>();
  if (*abort) {  // a copy did not come: those under way land before shared memory is released
    const uint64_t t0 = timer_ns();
    while (timer_ns() - t0 < 200000) __nanosleep(1000);
    if (lane == 0) atomicCAS(a.status, 0, (int)kOpsTimeout);
  }
}

// ---- combine_rows and its gradient ---------------------------------------------------------------------------
constexpr int kJoinWarps = 8, kJoinThreads = 32 + 32 * kJoinWarps, kJoinMostTopk = 32;
constexpr uint32_t kJoinMostPiece = 16 * 32 * kJoinWarps;  // a 16-byte word per thread

// Warp 0 loads, a lane a piece of a row.  In the gradient piece 0 of a slot's pieces is dout's, and the pieces of a token follow
// one another in a CTA, which sums its weights' gradients.
template <typename T, bool BACKWARD, int KEEP>  // KEEP: weights' gradients that a thread holds, a multiple of 8
__global__ void __launch_bounds__(kJoinThreads, 1) combine_rows_bulk_kernel(const CombineRows c, const BulkArgs a) {
  using namespace sm100;
  constexpr int N = 16 / sizeof(T);
  extern __shared__ uint8_t bulk_shared[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(bulk_shared) + 127) & ~(uintptr_t)127);
  const uint32_t ring = smem_u32(smem), full = ring + kBulkRing, empty = full + 8 * kBulkSlots, summed = empty + 8 * kBulkSlots;
  __shared__ int abort_flag;
  __shared__ int s_place[kBulkSlots][kJoinMostTopk];
  __shared__ float s_weight[kBulkSlots][kJoinMostTopk];
  __shared__ uint32_t s_spare[kBulkSlots];  // BACKWARD: bit k: the row of this number is nobody's
  __shared__ float s_dot[BACKWARD ? kBulkTurns : 1][kJoinWarps][BACKWARD ? KEEP : 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < a.slots; ++s) {
      mbar_init(full + 8 * s, 1);
      mbar_init(empty + 8 * s, kJoinWarps);
    }
    for (int s = 0; s < kBulkTurns; ++s) mbar_init(summed + 8 * s, kJoinWarps);
    fence_barrier_init();
  }
  __syncthreads();
  wait_predecessors();
  allow_successor();
  volatile int* abort = &abort_flag;
  const int64_t n_rows = c.tokens * c.topk, row_bytes = (int64_t)c.cols * sizeof(T);
  // The CTA's units are tokens, all pieces of each, or (few tokens) single pieces.
  const int64_t each = a.whole ? a.pieces : 1, units = a.whole ? c.tokens : c.tokens * a.pieces;
  const int64_t my_units = (units - blockIdx.x + gridDim.x - 1) / gridDim.x;
  auto unit_at = [&](int64_t u, int64_t& token, int64_t& from) {
    const int64_t unit = blockIdx.x + u * gridDim.x;
    token = a.whole ? unit : unit / a.pieces;
    from = a.whole ? 0 : (unit - token * a.pieces) * a.piece;
  };
  auto bytes_at = [&](int64_t from) { return (uint32_t)min((int64_t)a.piece, row_bytes - from); };
  const bool load_rows = !BACKWARD || c.dweights != nullptr;
  if (warp == 0) {
    // Places and weights are fetched for as many units as the warp has lanes for, a batch ahead: beside a busy TMA an ordinary load
    // takes microseconds (fetched one piece ahead, combine_rows of 8192 x 8 rows of 7168 took 278 us).
    const int batch = 32 / c.topk;
    const int of = lane / c.topk, k = lane - of * c.topk;  // this lane's unit of a batch, and its choice
    int place = -1, source = 0, next_place = -1, next_source = 0;
    float weight = 1.f, next_weight = 1.f;
    auto fetch = [&](int64_t u) {
      next_place = -1, next_source = 0;
      if (u + of >= my_units || of >= batch) return;
      int64_t token, from;
      unit_at(u + of, token, from);
      next_place = c.place[token * c.topk + k];
      if (next_place >= n_rows) next_place = -1;
      if (c.weights != nullptr) next_weight = c.weights[token * c.topk + k];
      if (BACKWARD) next_source = c.source[token * c.topk + k];
    };
    fetch(0);
    int in_batch = batch - 1;
    uint32_t s = 0, ph = 1;
    for (int64_t u = 0; u < my_units; ++u) {
      if (++in_batch == batch) {
        in_batch = 0;
        place = next_place, source = next_source, weight = next_weight;
        fetch(u + batch);
      }
      const bool here = of == in_batch;
      const uint32_t there = __ballot_sync(0xffffffffu, here && place >= 0);
      const uint32_t spare = __ballot_sync(0xffffffffu, here && source < 0) >> (in_batch * c.topk);
      int64_t token, from;
      unit_at(u, token, from);
      bool ok = true;
      for (int64_t p = 0; p < each; ++p, from += a.piece) {
        if (!(ok = __all_sync(0xffffffffu, mbar_wait(empty + 8 * s, ph, abort, a.budget_ns)))) break;
        const uint32_t bytes = bytes_at(from);
        if (here) s_place[s][k] = place, s_weight[s][k] = weight;
        __syncwarp();
        if (lane == 0) {
          s_spare[s] = spare;
          mbar_expect_tx(full + 8 * s, ((load_rows ? __popc(there) : 0) + (BACKWARD ? 1 : 0)) * bytes);
        }
        __syncwarp();
        const uint32_t dst = ring + s * a.slot;
        if (BACKWARD && lane == 0) bulk_load(dst, static_cast<const T*>(c.dout) + token * c.dout_ld + from / (int64_t)sizeof(T), bytes, full + 8 * s);
        if (load_rows && here && place >= 0)
          bulk_load(dst + (k + (BACKWARD ? 1 : 0)) * a.piece, static_cast<const T*>(c.rows) + place * c.ld + from / (int64_t)sizeof(T), bytes, full + 8 * s);
        if (++s == (uint32_t)a.slots) s = 0, ph ^= 1;
      }
      if (!ok) break;
    }
  } else {
    const int at = (threadIdx.x - 32) * 16;
    float dot[KEEP];
#pragma unroll
    for (int k = 0; k < KEEP; ++k) dot[k] = 0.f;
    uint32_t turn = 0, s = 0, ph = 0;
    const int64_t mine = my_units * each;
    int64_t token = 0, from = 0;
    for (int64_t n = 0, p = 0, u = 0; n < mine; ++n, from += a.piece) {
      if (p == 0) unit_at(u++, token, from);
      p = p + 1 < each ? p + 1 : 0;
      const uint32_t bytes = bytes_at(from);
      if (!__all_sync(0xffffffffu, mbar_wait(full + 8 * s, ph, abort, a.budget_ns))) break;
      const uint8_t* piece = smem + s * a.slot + at;
      const bool inside = at < (int)bytes;
      auto read = [&](int k, float (&f)[N]) {
        const uint4 raw = *reinterpret_cast<const uint4*>(piece + k * a.piece);
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (sizeof(T) == 4) {
            f[i] = __uint_as_float(w[i]);
          } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
            f[2 * i] = __uint_as_float(w[i] << 16), f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
          } else {
            const float2 two = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            f[2 * i] = two.x, f[2 * i + 1] = two.y;
          }
        }
      };
      auto write = [&](T* to, const float (&f)[N]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (sizeof(T) == 4) {
            w[i] = __float_as_uint(f[i]);
          } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
            const __nv_bfloat162 two = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&two);
          } else {
            const __half2 two = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&two);
          }
        }
        *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
      };
      const int64_t column = (from + at) / (int64_t)sizeof(T);
      if constexpr (!BACKWARD) {
        if (inside) {
          float sum[N];
#pragma unroll
          for (int i = 0; i < N; ++i) sum[i] = 0.f;
#pragma unroll 4
          for (int k = 0; k < c.topk; ++k) {
            if (s_place[s][k] < 0) continue;
            const float w = s_weight[s][k];
            float f[N];
            read(k, f);
#pragma unroll
            for (int i = 0; i < N; ++i) sum[i] = fmaf(w, f[i], sum[i]);
          }
          write(static_cast<T*>(c.out) + token * c.cols + column, sum);
        }
      } else {
        if (inside) {
          float d[N];
          read(0, d);
#pragma unroll
          for (int k = 0; k < KEEP; ++k) {
            if (k >= c.topk) continue;
            const int place = s_place[s][k];
            if (place >= 0) {
              if (c.dweights != nullptr) {
                float f[N];
                read(1 + k, f);
#pragma unroll
                for (int i = 0; i < N; ++i) dot[k] = fmaf(d[i], f[i], dot[k]);
              }
              if (c.drows != nullptr) {
                const float w = s_weight[s][k];
                float f[N];
#pragma unroll
                for (int i = 0; i < N; ++i) f[i] = w * d[i];
                write(static_cast<T*>(c.drows) + (int64_t)place * c.cols + column, f);
              }
            }
          }
          if (c.drows != nullptr && s_spare[s] != 0) {  // rows that nobody has
            float f[N];
#pragma unroll
            for (int i = 0; i < N; ++i) f[i] = 0.f;
            for (int k = 0; k < c.topk; ++k)
              if (s_spare[s] >> k & 1) write(static_cast<T*>(c.drows) + (token * c.topk + k) * c.cols + column, f);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty + 8 * s);
      if (++s == (uint32_t)a.slots) s = 0, ph ^= 1;
      if constexpr (BACKWARD) {
        if (from + a.piece < row_bytes || c.dweights == nullptr) continue;
        // the token's last piece: its weights' gradients, summed over the threads
#pragma unroll
        for (int k = 0; k < KEEP; ++k) {
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) dot[k] += __shfl_xor_sync(0xffffffffu, dot[k], o);
          if (lane == 0) s_dot[turn % kBulkTurns][warp - 1][k] = dot[k];
          dot[k] = 0.f;
        }
        // The first of the warps adds up.  The others go on: by the time that one of them is back at this turn, a slot has been
        // loaded again that the first warp gave up after reading the sums.
        const uint32_t bar = summed + 8 * (turn % kBulkTurns);
        if (lane == 0) mbar_arrive(bar);
        if (warp == 1) {
          if (!__all_sync(0xffffffffu, mbar_wait(bar, turn / kBulkTurns & 1, abort, a.budget_ns))) break;
          if (lane < c.topk) {
            float sum = 0.f;
#pragma unroll
            for (int w = 0; w < kJoinWarps; ++w) sum += s_dot[turn % kBulkTurns][w][lane];
            c.dweights[token * c.topk + lane] = sum;
          }
          __syncwarp();
        }
        ++turn;
      }
    }
  }
  __syncthreads();
  if (*abort) {
    const uint64_t t0 = timer_ns();
    while (timer_ns() - t0 < 200000) __nanosleep(1000);
    if (threadIdx.x == 0) atomicCAS(a.status, 0, (int)kOpsTimeout);
  }
}

}  // namespace ops
}  // namespace lplb

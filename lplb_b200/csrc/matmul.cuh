// Products in 16 bits with an epilogue, and their gradients, on the tensor cores: accumulators in tensor memory, operands staged by
// TMA into 128-byte-swizzled shared memory.
//
//   forward   z = a b^T + bias, out = act(z) + residual     a [m, k], b [n, k]
//   input     da = dz b                                     dz [m, n]
//   weight    db = dz^T a
//
// Every one is D[i, j] = sum over r of P[i, r] Q[j, r] with i along the result's rows in memory (neighbouring values) and j from row to
// row: P is the operand that holds `features`, Q the one that holds result rows.
//
//               P                  Q                r
//   forward     b, K-major         a, K-major       k
//   input       b, MN-major        dz, K-major      n
//   weight      a, MN-major        dz, MN-major     rows of the group
//
// MN-major operands are read as they lie in memory: nothing is transposed on the way.  P is on the tensor core's M side (256 a
// pair of CTAs), Q on its N side, where a tile takes any multiple of 32 rows: the number of rows of a group is arbitrary.
//
// With groups the tiles go group by group.  A weight tile sums over its group's rows alone: its last block of 64 rows is fetched in
// boxes of 16, 8, 4, 2 and 1 rows, and what is missing of the last 16 is fetched from behind the tensor's last row, where TMA
// fills in zeros, so that nothing of the next group (an infinity times zero) comes in.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"
#include "matmul_api.h"
#include "tcgen05.cuh"

namespace lplb {
namespace ops {

// ---- the epilogue ------------------------------------------------------------------------------------
struct Epilogue {
  const void* bias;
  const void* residual;
  void* out;
  void* pre;
  int64_t residual_ld, out_ld, pre_ld;
  int n;            // features: weight rows, the length of a bias row
  int activation;
  Type type, bias_type;  // of out, residual and pre; of the bias
};

__device__ __forceinline__ float load_as_float(const void* p, Type type, int64_t i) {
  if (type == Type::kF32) return static_cast<const float*>(p)[i];
  if (type == Type::kBf16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store_float(void* p, Type type, int64_t i, float v) {
  if (type == Type::kF32) static_cast<float*>(p)[i] = v;
  else if (type == Type::kBf16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else static_cast<__half*>(p)[i] = __float2half_rn(v);
}
// Four values that are `S` apart; next to one another (S = 1) they start on a boundary of their size and go in one piece.
template <int S>
__device__ __forceinline__ void load4(const void* p, Type type, int64_t i, int limit, float (&v)[4]) {
  if constexpr (S == 1) {
    if (limit <= 0) return;
    if (type == Type::kF32) {
      const float4 f = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
      v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
      return;
    }
    const uint2 raw = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i);
    const uint32_t w[2] = {raw.x, raw.y};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (type == Type::kBf16) {
        v[2 * h] = __uint_as_float(w[h] << 16), v[2 * h + 1] = __uint_as_float(w[h] & 0xFFFF0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[h]));
        v[2 * h] = f.x, v[2 * h + 1] = f.y;
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j * S < limit) v[j] = load_as_float(p, type, i + j * S);
  }
}
template <int S>
__device__ __forceinline__ void store4(void* p, Type type, int64_t i, int limit, const float (&v)[4]) {
  if constexpr (S == 1) {
    if (limit <= 0) return;
    if (type == Type::kF32) {
      *reinterpret_cast<float4*>(static_cast<float*>(p) + i) = make_float4(v[0], v[1], v[2], v[3]);
      return;
    }
    uint2 raw;
    if (type == Type::kBf16) {
      const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
      raw = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    } else {
      const __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
      raw = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    }
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p) + i) = raw;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j * S < limit) store_float(p, type, i + j * S, v[j]);
  }
}

// (__expf is off by 2 + 1.2 |x| units in the last place, the quotient by two: 2^-20 of the value where it matters, and the
// result, of up to 24 bits, is mostly rounded to 8 or 11)
__device__ __forceinline__ float sigmoid_of(float z) { return __fdividef(1.f, 1.f + __expf(-z)); }
__device__ __forceinline__ float activated(float z, int activation) {
  if (activation == kSilu) return z * sigmoid_of(z);
  if (activation == kGelu) return z * normcdff(z);
  if (activation == kRelu) return z < 0.f ? 0.f : z;  // NaN stays
  return z;
}

// One CTA's 128 weight rows as columns of the result.  Four columns of a thread: `column`, and S apart.
// GATED: 64 gate rows and their 64 up rows, 64 columns of the result.
template <int S, bool GATED>
struct Columns {
  int64_t bias_row;  // first value of the group's bias
  int out, gate;     // first column in out and residual; in bias and pre (GATED: its up column is kGateBlock behind)
  int limit;         // of the four, those with S * j below this are there
  float bias[4], up_bias[4];
  __device__ __forceinline__ void load_bias(const Epilogue& e, int group) {
#pragma unroll
    for (int j = 0; j < 4; ++j) bias[j] = up_bias[j] = 0.f;
    if (e.bias == nullptr) return;
    const int64_t at = (int64_t)group * e.n + gate;
    load4<S>(e.bias, e.bias_type, at, limit, bias);
    if (GATED) load4<S>(e.bias, e.bias_type, at + kGateBlock, limit, up_bias);
  }
  // z (and up): sums without the bias, of result row `row`; r: the residual's values
  __device__ __forceinline__ void finish(const Epilogue& e, int64_t row, float (&z)[4], float (&up)[4], const float (&r)[4]) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) z[j] += bias[j];
    if (GATED) {
#pragma unroll
      for (int j = 0; j < 4; ++j) up[j] += up_bias[j];
    }
    if (e.pre != nullptr) {
      store4<S>(e.pre, e.type, row * e.pre_ld + gate, limit, z);
      if (GATED) store4<S>(e.pre, e.type, row * e.pre_ld + gate + kGateBlock, limit, up);
    }
    if (GATED) {
#pragma unroll
      for (int j = 0; j < 4; ++j) z[j] = z[j] * sigmoid_of(z[j]) * up[j];
    } else if (e.activation != kNoActivation) {
#pragma unroll
      for (int j = 0; j < 4; ++j) z[j] = activated(z[j], e.activation);
    }
    if (e.residual != nullptr) {
#pragma unroll
      for (int j = 0; j < 4; ++j) z[j] += r[j];
    }
    store4<S>(e.out, e.type, row * e.out_ld + out, limit, z);
  }
  __device__ __forceinline__ void load_residual(const Epilogue& e, int64_t row, float (&r)[4]) const {
    if (e.residual != nullptr) load4<S>(e.residual, e.type, row * e.residual_ld + out, limit, r);
  }
};

// ---- CTA pairs: tiles of 256 features x up to 256 result rows ---------------------------------------------
enum Mode : int { kForward = 0, kForwardGated = 1, kInput = 2, kWeight = 3 };

constexpr int kPairM = 256, kPairN = 256, kPairK = 64, kHalfM = kPairM / 2;
constexpr int kRowStep = 32;      // result rows of a tile come in these
constexpr int kWeightStep = 128;  // kWeight: whole chunks of 64 for either CTA
constexpr int kChunk = 64;        // values of an MN-major operand in one swizzled row
constexpr uint32_t kChunkBytes = kChunk * kPairK * 2;
constexpr int kBoxes = 6;         // K-major: 128, 64, 32, 16 result rows; kWeight: 64, 16, 8, 4, 2, 1 rows of the sum
constexpr uint32_t kStageP = kHalfM * kPairK * 2;
constexpr uint32_t kPairRing = 192 * 1024;
constexpr int kPairStages = 11;
constexpr int kTurnRows = 16;     // result rows that go through shared memory at a time
constexpr uint32_t kTurn = kTurnRows * kHalfM * 4;
constexpr uint32_t kPairBars = 256;
constexpr size_t kPairSmem = 1024 + kPairRing + kPairBars + 2 * kTurn;
constexpr int kPairThreads = 192, kPairColumns = 512;

struct PairMaps {
  CUtensorMap p[kBoxes], q[kBoxes];  // K-major P: the first only
};
struct PairArgs {
  const int* rows;  // [groups] or null
  int groups;
  int n_rows;       // m
  int features;     // i: n (kForward), k (kInput, kWeight)
  int result_rows;  // kWeight: n, rows of a group's result
  int k_blocks;     // blocks of r; kWeight: of the group's rows
  int tiles_p;      // ceil(features / 256)
  int tile_steps;   // result rows of a tile at most, in steps
  int wide;         // four neighbouring values of everything in the epilogue start on a boundary of their size
  uint32_t idesc;
  int* status;
  unsigned long long budget_ns;
  Epilogue e;
};

// The tile list: group by group, in a group the tiles of P one after the other and in each the result rows, split evenly.
template <Mode MODE>
struct PairTile {
  int group = 0, first = 0;  // first tile of the group
  int p = 0, row0 = 0, n = 0;
  static constexpr int kStep = MODE == kWeight ? kWeightStep : kRowStep;
  __device__ __forceinline__ bool seek(int t, const int* rows, const PairArgs& a) {
    for (; group < a.groups; ++group) {
      const int high = MODE == kWeight ? (rows[group] > 0 ? a.result_rows : 0) : rows[group];
      const int steps = (high + kStep - 1) / kStep, tiles = (steps + a.tile_steps - 1) / a.tile_steps;
      if (t < first + tiles * a.tiles_p) {
        const int local = t - first;
        p = local / tiles;
        const int i = local - p * tiles, base = steps / tiles, extra = steps - base * tiles;
        row0 = (i * base + min(i, extra)) * kStep;
        n = (base + (i < extra)) * kStep;
        return true;
      }
      first += tiles * a.tiles_p;
    }
    return false;
  }
};

// Roles: warp 0 TMA, warp 1 tensor memory and (in the pair's first CTA) matrix instructions, warps 2-5 epilogue.  Two accumulators:
// the epilogue of a tile runs beside the sums of the next.
template <Mode MODE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
pair_matmul_kernel(const __grid_constant__ PairMaps maps, const PairArgs a) {
  using namespace sm100;
  constexpr bool kGated = MODE == kForwardGated, kPmn = MODE >= kInput, kQmn = MODE == kWeight;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kPairRing);
  float* turns = reinterpret_cast<float*>(smem + kPairRing + kPairBars);
  const uint32_t bar_full = smem_u32(bars), bar_empty = smem_u32(bars + kPairStages);
  const uint32_t bar_tfull = smem_u32(bars + 2 * kPairStages), bar_tempty = smem_u32(bars + 2 * kPairStages + 2);
  static_assert((2 * kPairStages + 4) * 8 <= kPairBars, "barriers");
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  __shared__ int s_rows[kMatmulMaxGroups], s_start[kMatmulMaxGroups + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int half = (int)cluster_cta_rank();
  const int n_pairs = (int)gridDim.x / 2, pair = (int)blockIdx.x / 2;
  allow_successor();
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < kPairStages; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar_tfull + 8 * b, 1);
      mbar_init(bar_tempty + 8 * b, 8);  // four epilogue warps of either CTA
    }
    fence_barrier_init();
    tma_prefetch_desc(&maps.p[0]);
    tma_prefetch_desc(&maps.q[0]);
  }
  if (warp == 1) tmem_alloc(smem_u32(&tmem_slot), kPairColumns);
  wait_predecessors();
  if (warp == 2) {  // groups one after the other, none beyond the last row
    long long before = 0;
    for (int e0 = 0; e0 < a.groups; e0 += 32) {
      const int e = e0 + lane;
      const long long mine = e >= a.groups ? 0 : a.rows != nullptr ? max(a.rows[e], 0) : a.n_rows;
      long long scan = mine;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, scan, d);
        if (lane >= d) scan += v;
      }
      if (e < a.groups) {
        const int from = (int)min((long long)a.n_rows, before + scan - mine), to = (int)min((long long)a.n_rows, before + scan);
        s_rows[e] = to - from;
        s_start[e] = from;
        s_start[e + 1] = to;  // (also written, the same, by the next lane)
      }
      before += __shfl_sync(0xffffffffu, scan, 31);
      __syncwarp();
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync();  // the peer's barriers are initialised and its tensor memory is allocated
  tc_fence_after_sync();
  const uint32_t tmem_base = tmem_slot;
  volatile int* abort = &abort_flag;
  const uint64_t budget = a.budget_ns;
  PairTile<MODE> cur;
  // a stage holds P and as many result rows as the launch's largest tile stages per CTA
  int largest = 1;
  for (int e = lane; e < a.groups; e += 32) {
    const int high = MODE == kWeight ? a.result_rows : s_rows[e];
    const int steps = (high + cur.kStep - 1) / cur.kStep, tiles = (steps + a.tile_steps - 1) / a.tile_steps;
    if (tiles > 0) largest = max(largest, (steps + tiles - 1) / tiles);
  }
  largest = __reduce_max_sync(0xffffffffu, largest);
  const uint32_t stage_bytes = kStageP + largest * (cur.kStep / 2) * kPairK * 2;
  const uint32_t stages = min((uint32_t)kPairStages, kPairRing / stage_bytes);
  auto find = [&](uint32_t i) { return cur.seek(pair + (int)i * n_pairs, s_rows, a); };
  auto blocks_of = [&]() { return MODE == kWeight ? (s_rows[cur.group] + kPairK - 1) / kPairK : a.k_blocks; };
  // kWeight: rows of block kb, rounded up to a matrix instruction's 16
  auto rows_of = [&](int kb) { return MODE == kWeight ? min(kPairK, s_rows[cur.group] - kb * kPairK) : kPairK; };

  if (warp == 0) {
    // ---------------- TMA ----------------
    if (elect_one()) {
      const uint32_t lead_full = map_to_rank(bar_full, 0);
      uint32_t s = 0, ph = 0;
      for (uint32_t i = 0; find(i) && !*abort; ++i) {
        const int mine = cur.n / 2;
        const int feature = cur.p * kPairM + half * kHalfM;
        const int row = (MODE == kWeight ? 0 : s_start[cur.group]) + cur.row0 + half * mine;
        const int blocks = blocks_of();
        for (int kb = 0; kb < blocks; ++kb) {
          if (!mbar_wait(bar_empty + 8 * s, ph ^ 1, abort, budget)) break;
          const uint32_t full = lead_full + 8 * s;
          const int there = rows_of(kb), deep = (there + 15) / 16 * 16;
          if (half == 0) mbar_expect_tx(bar_full + 8 * s, 2 * (uint32_t)(kHalfM + mine) * (uint32_t)deep * 2);
          uint32_t dst = smem_u32(smem) + s * stage_bytes;
          if constexpr (MODE == kForward) {
            tma_pair_load_3d(dst, &maps.p[0], full, kb * kPairK, feature, cur.group);
          } else if constexpr (MODE == kForwardGated) {
            tma_pair_load_5d(dst, &maps.p[0], full, kb * kPairK, half * (kHalfM / 32), cur.group * a.tiles_p + cur.p);
          } else if constexpr (MODE == kInput) {
            for (int c = 0; c < kHalfM / kChunk; ++c)
              tma_pair_load_3d(dst + c * kChunkBytes, &maps.p[0], full, feature + c * kChunk, kb * kPairK, cur.group);
          }
          if constexpr (MODE != kWeight) {
            dst += kStageP;
            int r = row;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
              const int n = kPairN / 2 >> b;
              if (mine & n) {
                tma_pair_load_2d(dst, &maps.q[b], full, kb * kPairK, r);
                dst += n * kPairK * 2;
                r += n;
              }
            }
          } else {
            const int from = s_start[cur.group] + kb * kPairK;
            auto chunk = [&](uint32_t to, const CUtensorMap* map, int x) {
              if (there == kPairK) {
                tma_pair_load_2d(to, &map[0], full, x, from);
                return;
              }
              int at = 0;
              auto box = [&](int b, int n, int y) {
                tma_pair_load_2d(to + at * 128, &map[b], full, x, y);
                at += n;
              };
              while (at + 16 <= there) box(1, 16, from + at);
#pragma unroll
              for (int b = 2; b < kBoxes; ++b)
                if ((there & 15) & (32 >> b)) box(b, 32 >> b, from + at);
              const int missing = deep - there;
#pragma unroll
              for (int b = kBoxes - 1; b >= 2; --b)  // the smallest first: every box starts on a multiple of its size
                if (missing & (32 >> b)) box(b, 32 >> b, a.n_rows);
            };
            for (int c = 0; c < kHalfM / kChunk; ++c) chunk(dst + c * kChunkBytes, maps.p, feature + c * kChunk);
            dst += kStageP;
            for (int c = 0; c < mine / kChunk; ++c) chunk(dst + c * kChunkBytes, maps.q, row + c * kChunk);
          }
          if (++s == stages) s = 0, ph ^= 1;
        }
      }
    }
  } else if (warp == 1) {
    // ---------------- matrix instructions, for both CTAs ----------------
    if (half == 0 && elect_one()) {
      uint32_t s = 0, ph = 0;
      for (uint32_t i = 0; find(i) && !*abort; ++i) {
        const uint32_t acc = i & 1, acc_ph = (i >> 1) & 1;
        if (!mbar_wait(bar_tempty + 8 * acc, acc_ph ^ 1, abort, budget)) break;
        tc_fence_after_sync();
        const uint32_t idesc = a.idesc | umma_idesc_size(kPairM, cur.n), tmem_d = tmem_base + acc * kPairN;
        const int blocks = blocks_of();
        bool ok = true;
        for (int kb = 0; kb < blocks; ++kb) {
          if (!mbar_wait(bar_full + 8 * s, ph, abort, budget)) {
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t base = smem_u32(smem) + s * stage_bytes;
          const uint64_t dp = kPmn ? umma_desc_mn_sw128(base, kChunkBytes) : umma_desc_sw128(base);
          const uint64_t dq = kQmn ? umma_desc_mn_sw128(base + kStageP, kChunkBytes) : umma_desc_sw128(base + kStageP);
          const int steps = (rows_of(kb) + 15) / 16;
#pragma unroll
          for (int k = 0; k < kPairK / 16; ++k)  // 16 of the sum: 32 bytes of a K-major row, 16 rows of an MN-major chunk
            if (k < steps) umma_pair_bf16(tmem_d, dp + k * (kPmn ? 2048 >> 4 : 2), dq + k * (kQmn ? 2048 >> 4 : 2), idesc, (kb | k) != 0);
          umma_pair_commit(bar_empty + 8 * s);
          if (++s == stages) s = 0, ph ^= 1;
        }
        if (!ok) break;
        umma_pair_commit(bar_tfull + 8 * acc);
      }
    }
  } else {
    // ---------------- epilogue ----------------
    const int quarter = warp & 3;  // the tensor memory lanes that this warp may read
    const int ew = warp - 2, et = threadIdx.x - 64;
    const Epilogue& e = a.e;
    // What has no product: rows behind the last group, matrices without rows.  (The first tile's sums are under way meanwhile.)
    const int64_t cta = blockIdx.x, ctas = gridDim.x;
    const int out_cols = kGated ? a.features / 2 : a.features;
    auto clear_row = [&](int64_t row) {
      if (a.wide) {
        for (int c = 4 * et; c < out_cols; c += 512) {
          float v[4] = {0.f, 0.f, 0.f, 0.f};
          if (e.residual != nullptr) load4<1>(e.residual, e.type, row * e.residual_ld + c, 4, v);
          store4<1>(e.out, e.type, row * e.out_ld + c, 4, v);
        }
      } else {
        for (int c = et; c < out_cols; c += 128)
          store_float(e.out, e.type, row * e.out_ld + c, e.residual != nullptr ? load_as_float(e.residual, e.type, row * e.residual_ld + c) : 0.f);
      }
    };
    if constexpr (MODE == kWeight) {
      for (int g = 0; g < a.groups; ++g)
        if (s_rows[g] == 0)
          for (int64_t r = cta; r < a.result_rows; r += ctas) clear_row((int64_t)g * a.result_rows + r);
    } else {
      for (int64_t r = s_start[a.groups] + cta; r < a.n_rows; r += ctas) clear_row(r);
    }
    uint32_t turn = 0;
    auto tiles = [&](auto wide) {
      constexpr bool kWide = decltype(wide)::value;
      constexpr int kLanes = kGated ? 16 : 32;              // that share a row of 64 or 128 columns
      constexpr int S = kWide ? 1 : kLanes;
      constexpr int kPer = kTurnRows * kLanes / 128;        // rows of a turn per thread
      const int in_row = lane & (kLanes - 1);
      const int f = kWide ? 4 * in_row : in_row;            // first of the thread's four columns, of the CTA's
      const int row_of = ew * (32 / kLanes) + lane / kLanes;  // its first row of a turn; the next are 128 / kLanes behind
      for (uint32_t i = 0;; ++i) {
        // All four warps leave together: they meet at barriers, and tcgen05.ld is a whole-warp instruction.
        if (!epilogue_all(find(i) && !*abort)) break;
        const uint32_t acc = i & 1, acc_ph = (i >> 1) & 1;
        const int left = (MODE == kWeight ? a.result_rows : s_rows[cur.group]) - cur.row0, n = min(cur.n, left);
        const int64_t row0 = (MODE == kWeight ? (int64_t)cur.group * a.result_rows : (int64_t)s_start[cur.group]) + cur.row0;
        Columns<S, kGated> mine;
        if constexpr (kGated) {
          mine.out = cur.p * kHalfM + half * (kHalfM / 2) + f;
          mine.gate = cur.p * kPairM + half * (kHalfM / 2) + f;
          mine.limit = kHalfM;  // whole blocks
        } else {
          mine.out = mine.gate = cur.p * kPairM + half * kHalfM + f;
          mine.limit = a.features - mine.out;
        }
        mine.load_bias(e, cur.group);
        if (!epilogue_all(mbar_wait(bar_tfull + 8 * acc, acc_ph, abort, budget))) break;
        tc_fence_after_sync();
        const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + acc * kPairN;
        for (int c0 = 0; c0 < n; c0 += kTurnRows, turn ^= 1) {
          float* stage = turns + turn * (kTurnRows * kHalfM);
          float r[kPer][4];
#pragma unroll
          for (int q = 0; q < kPer; ++q) {
            const int at = c0 + row_of + q * (128 / kLanes);
            if (at < n) mine.load_residual(e, row0 + at, r[q]);
          }
          float v[16];
          __syncwarp();
          tmem_ld_32x16(taddr + c0, v);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 16; ++j) stage[j * kHalfM + quarter * 32 + lane] = v[j];
          epilogue_sync();
#pragma unroll
          for (int q = 0; q < kPer; ++q) {
            const int in_turn = row_of + q * (128 / kLanes), at = c0 + in_turn;
            if (at >= n) continue;
            const float* from = stage + in_turn * kHalfM;
            float z[4], up[4];
            // a warp's 32 lanes of tensor memory are, gated, 16 gate rows and their 16 up rows
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int c = f + j * S;
              z[j] = from[kGated ? (c >> 4) * 32 + (c & 15) : c];
              up[j] = kGated ? from[(c >> 4) * 32 + 16 + (c & 15)] : 0.f;
            }
            mine.finish(e, row0 + at, z, up, r[q]);
          }
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive_remote(map_to_rank(bar_tempty + 8 * acc, 0));
      }
    };
    if (a.wide) tiles(std::true_type{});
    else tiles(std::false_type{});
  }

  // ---------------- teardown ----------------
  if (*abort) {  // a role gave up: copies in flight land before shared and tensor memory are released
    const uint64_t t0 = timer_ns();
    while (timer_ns() - t0 < 200000) __nanosleep(1000);
    if (threadIdx.x == 0) atomicCAS(a.status, 0, (int)kOpsTimeout);
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync();  // neither CTA leaves while the other may still signal it or read its operands
  if (warp == 1) tmem_dealloc(tmem_base, kPairColumns);
}

}  // namespace ops
}  // namespace lplb

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
// With groups the tiles go group by group.  A weight tile sums over its group's rows alone, and nothing of the next group (an infinity
// times zero) may come in: a group's last block of 64 rows, where it is not whole, is copied beforehand, with zeros behind it up to the
// 16 rows of a matrix instruction.  (Fetched in boxes of 16, 8, 4, 2 and 1 rows, the rest from behind the tensor's last row, where TMA
// fills in zeros, such a block cost 1.5 to 3 us of a tile's 7: issuing a box takes the producer some 100 cycles whatever its size.  So a
// box also holds both chunks of 64 columns that a CTA has, where it can.)
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
  const uint32_t* most;  // of the gradients: magnitudes that say which part of a power of two a result row's sums are, or null
  int64_t residual_ld, out_ld, pre_ld;
  int n;            // features: weight rows, the length of a bias row
  int activation;
  Type type, bias_type;  // of out and residual; of the bias.  pre is in 32 bits: what is rounded there comes back in every gradient
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
// dz in float16: values up to 2^127 and down to 2^-149 would be infinite and zero there, and with them a gradient that is neither.  So they
// are stored times 2^(14 - e) for a largest finite magnitude of 2^e (the products see 2^14 to 2^15 at most), and the sums multiplied by
// 2^(e - 14) before they are rounded.  Both are exact; what lies 2^28 below the largest has fewer bits, an error of 2^-39 of the largest.
__device__ __forceinline__ uint32_t part_exponent(uint32_t most) { return max(most >> 23, 15u); }  // both factors are normal numbers
__device__ __forceinline__ float part_of(uint32_t most) { return __uint_as_float((268u - part_exponent(most)) << 23); }
__device__ __forceinline__ float whole_of(uint32_t most) { return __uint_as_float((part_exponent(most) - 14u) << 23); }
__device__ __forceinline__ uint32_t finite_magnitude(float v) {
  const uint32_t b = __float_as_uint(v) & 0x7FFFFFFFu;
  return b < 0x7F800000u ? b : 0u;
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

// (__expf is off by 2 + 1.2 |z| units in the last place, the quotient by two: some |z| units come from z's own last bit, too.  Below z = -87, where
// silu is 1e-36, it is 0.)
__device__ __forceinline__ float sigmoid_of(float z) { return __fdividef(1.f, 1.f + __expf(-z)); }
// The normal distribution's function, and e^(-z^2 / 2), in few instructions and good to some 2^-20 of the value on either side: for
// u >= 0 Phi(-u) e^(u^2 / 2) is smooth and falls slowly, here as a polynomial in 1 / (1 + 0.4 u), fitted to 0 <= u <= 14 by least
// squares of the relative error with weights that level it (8e-8; in 32 bits 3.5e-7).  us, 4096 x 4096 x 1024 in bf16 with gelu: this
// 38, 0.5 erfc(-z / sqrt 2) 55, 0.5 + 0.5 erf(z / sqrt 2) 39, but that is off by 2^-24, not of the value: 4 % at z = -5.
__device__ __forceinline__ float normal_cdf(float z, float& bell) {
  constexpr float kCoefficients[] = {-0.0396009646f, 0.20060125f,  -0.373683333f, 0.250973463f,    -0.0123857474f,
                                     0.158416525f,   0.155786633f, 0.159904182f,  -1.19874376e-05f};
  const float t = __fdividef(1.f, fmaf(0.4f, fabsf(z), 1.f));
  bell = __expf(__fmul_rn(-0.5f, __fmul_rn(z, z)));
  float q = kCoefficients[0];
#pragma unroll
  for (int i = 1; i < 9; ++i) q = fmaf(q, t, kCoefficients[i]);
  q = __fmul_rn(q, bell);
  return z > 0.f ? __fsub_rn(1.f, q) : q;
}
// (Which activation is asked once for all values: asked for each, 4096 x 4096 x 1024 with silu took 65 us, without an activation 25.  Values are
// rounded by themselves, not fused with what is added to them: every path of a product has the same bits.)
template <int N>
__device__ __forceinline__ void activate(float (&z)[N], int activation) {
  if (activation == kSilu) {
#pragma unroll
    for (int j = 0; j < N; ++j) z[j] = __fmul_rn(z[j], sigmoid_of(z[j]));
  } else if (activation == kGelu) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      float bell;
      z[j] = __fmul_rn(z[j], normal_cdf(z[j], bell));
    }
  } else if (activation == kRelu) {
#pragma unroll
    for (int j = 0; j < N; ++j) z[j] = z[j] < 0.f ? 0.f : z[j];  // NaN stays
  }
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
      store4<S>(e.pre, Type::kF32, row * e.pre_ld + gate, limit, z);
      if (GATED) store4<S>(e.pre, Type::kF32, row * e.pre_ld + gate + kGateBlock, limit, up);
    }
    if (GATED) {
#pragma unroll
      for (int j = 0; j < 4; ++j) z[j] = __fmul_rn(__fmul_rn(z[j], sigmoid_of(z[j])), up[j]);
    } else {
      activate(z, e.activation);
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

// 32 bytes, on a boundary of 32, in one piece: a whole sector.
__device__ __forceinline__ void st_global_v8(void* p, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
               ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

// ---- CTA pairs: tiles of 256 features x up to 256 result rows ---------------------------------------------
enum Mode : int { kForward = 0, kForwardGated = 1, kInput = 2, kWeight = 3 };

constexpr int kPairM = 256, kPairN = 256, kPairK = 64, kHalfM = kPairM / 2;
constexpr int kRowStep = 32;      // result rows of a tile come in these
constexpr int kWeightStep = 128;  // kWeight: whole chunks of 64 for either CTA
constexpr int kChunk = 64;        // values of an MN-major operand in one swizzled row
constexpr uint32_t kChunkBytes = kChunk * kPairK * 2;
constexpr int kBoxes = 4;         // K-major Q: 128, 64, 32, 16 result rows; kWeight: 64 rows of the sum, of a group's copy
constexpr uint32_t kStageP = kHalfM * kPairK * 2;
constexpr uint32_t kPairRing = 192 * 1024;
constexpr int kPairStages = 11;
constexpr int kStoreWarps = 8;      // of the epilogue: two for every quarter of tensor memory's lanes
constexpr uint32_t kTurn = 2048;   // of one such warp: 32 features x 32 result rows in 16 bits, or x 16 in 32
constexpr uint32_t kPairBars = 256;
constexpr size_t kPairSmem = 1024 + kPairRing + kPairBars + kStoreWarps * kTurn;
constexpr int kPairThreads = 64 + 32 * kStoreWarps, kPairColumns = 512;
// The tensor cores cut an accumulator's last bits off at every addition, which makes a long sum too small: one of products of the same sign by
// 6e-9 of it per product (3e-6 over 512, 1.0e-4 over 16,384, 6.7e-3 over 2^20, measured), one of either sign less, 7e-6 over 7168, where sums in 32
// bits that are rounded are off by 1e-6.  A result in 32 bits shows that, so its sum is taken over `kSumBlocks` blocks at a time in tensor
// memory, and these sums are added in registers (either sign: off by 5e-7 whatever the length).  A result in 16 bits hides it behind its
// rounding up to `longest_part` products; of longer sums the parts are added in tensor memory, in the accumulator that is not summed into.
// Tiles of at most `kSumRows` result rows: a thread holds half of them.  8192 x 4096 x 7168 in 450-500 us (16 bits 340-370),
// 1001 x 4100 x 2064 in 24.3 (20.7); blocks of 4 541 and 25.9; 192 rows, whose sums do not fit the registers, 612 and 37.8.
constexpr int kSumBlocks = 8, kSumRows = 128;
// Products of one accumulator for a result of the type: what is cut off is at most a tenth of half a step (2^-11 and 2^-8).  It also keeps the
// epilogue's wait for a sum far below its limit.
constexpr int longest_part(Type type) { return type == Type::kF32 ? kSumBlocks * kPairK : type == Type::kF16 ? 8192 : 65536; }

struct PairMaps {
  CUtensorMap p[2], q[kBoxes];  // P: the first only, but for kWeight
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
  int p_chunks, q_chunks;  // chunks of an MN-major operand that a box holds: 2 where columns come in whole chunks (q: and a CTA has two)
  int copies;       // kWeight: the last blocks of groups have been copied
  int part_blocks;  // of a sum, for one accumulator
  int wide;         // four neighbouring values of everything in the epilogue start on a boundary of their size
  int plain;        // a result in 16 bits, rows (the residual's too) of whole 16-byte words on boundaries
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

// Roles: warp 0 TMA, warp 1 tensor memory and (in the pair's first CTA) matrix instructions, warps 2-9 epilogue, every one by itself:
// it turns 32 features x 32 result rows round in shared memory of its own.  Two accumulators: the epilogue of a tile runs beside the
// sums of the next.  (With four warps that met at a barrier every 16 rows a weight's gradient of 32 experts, 512 rows each on average,
// 4096 x 7168, took 3070 us: its tiles have 8 blocks to sum, and 1750 cycles went into every 16 rows.)
// Of a sum that is longer than one part the parts come one after the other in the tile's accumulator, and their sum stays in the other one, of
// which every epilogue warp reads and writes what is its own alone.  So the tiles keep their height: the input's gradient of 1024 x 151936 x 4096
// takes 847 us in three parts, 844 in one, and in IN_32's way 1.5 times that.  IN_32, a result in 32 bits: parts so short
// that they alternate between the accumulators, and are added in registers.
template <Mode MODE, bool IN_32>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
pair_matmul_kernel(const __grid_constant__ PairMaps maps, const PairArgs a) {
  using namespace sm100;
  constexpr bool kGated = MODE == kForwardGated, kPmn = MODE >= kInput, kQmn = MODE == kWeight;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kPairRing);
  uint8_t* turns = smem + kPairRing + kPairBars;
  const uint32_t bar_full = smem_u32(bars), bar_empty = smem_u32(bars + kPairStages);
  const uint32_t bar_tfull = smem_u32(bars + 2 * kPairStages), bar_tempty = smem_u32(bars + 2 * kPairStages + 2);
  static_assert((2 * kPairStages + 4) * 8 <= kPairBars, "barriers");
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  __shared__ int s_rows[kMatmulMaxGroups], s_start[kMatmulMaxGroups + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int half = (int)cluster_cta_rank();
  const int n_pairs = (int)gridDim.x / 2, pair = (int)blockIdx.x / 2;
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < kPairStages; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar_tfull + 8 * b, 1);
      mbar_init(bar_tempty + 8 * b, 2 * kStoreWarps);  // of both CTAs
    }
    fence_barrier_init();
    tma_prefetch_desc(&maps.p[0]);
    tma_prefetch_desc(&maps.q[0]);
  }
  cluster_sync();  // both CTAs have begun
  if (warp == 1) tmem_alloc(smem_u32(&tmem_slot), kPairColumns);
  wait_predecessors();
  allow_successor();
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
  if (warp == 1) tmem_relinquish();
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
          const int there = rows_of(kb);
          if (half == 0) mbar_expect_tx(bar_full + 8 * s, 2 * (uint32_t)(kHalfM + mine) * kPairK * 2);
          uint32_t dst = smem_u32(smem) + s * stage_bytes;
          if constexpr (MODE == kForward) {
            tma_pair_load_3d(dst, &maps.p[0], full, kb * kPairK, feature, cur.group);
          } else if constexpr (MODE == kForwardGated) {
            tma_pair_load_5d(dst, &maps.p[0], full, kb * kPairK, half * (kHalfM / 32), cur.group * a.tiles_p + cur.p);
          } else if constexpr (MODE == kInput) {
            if (a.p_chunks == 2)
              tma_pair_load_4d(dst, &maps.p[0], full, kb * kPairK, feature / kChunk, cur.group);
            else
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
            // a group's last block, where it is not whole, from its copy
            const int from_copy = a.copies && there < kPairK;
            const int from = from_copy ? cur.group * kPairK : s_start[cur.group] + kb * kPairK;
            auto load = [&](uint32_t to, const CUtensorMap* map, int chunks, int x) {  // x: of the first column, a multiple of 64
              if (chunks == 2) tma_pair_load_3d(to, map, full, 0, from, x / kChunk);
              else tma_pair_load_2d(to, map, full, x, from);
            };
            for (int c = 0; c < kHalfM / kChunk; c += a.p_chunks) load(dst + c * kChunkBytes, &maps.p[from_copy], a.p_chunks, feature + c * kChunk);
            dst += kStageP;
            for (int c = 0; c < mine / kChunk; c += a.q_chunks) load(dst + c * kChunkBytes, &maps.q[from_copy], a.q_chunks, row + c * kChunk);
          }
          if (++s == stages) s = 0, ph ^= 1;
        }
      }
    }
  } else if (warp == 1) {
    // ---------------- matrix instructions, for both CTAs ----------------
    if (half == 0 && elect_one()) {
      uint32_t s = 0, ph = 0, acc = 0, used = 0;  // used: a bit per accumulator, turned over by every sum that is handed to the epilogue
      const int part_blocks = IN_32 ? kSumBlocks : a.part_blocks;
      for (uint32_t i = 0; find(i) && !*abort; ++i) {
        const uint32_t idesc = a.idesc | umma_idesc_size(kPairM, cur.n);
        const int blocks = blocks_of();
        bool ok = true;
        uint32_t tmem_d = 0;
        for (int kb = 0, in_part = 0; kb < blocks; ++kb) {
          const bool first = in_part == 0, last = kb == blocks - 1 || in_part == part_blocks - 1;
          in_part = last ? 0 : in_part + 1;
          if (first) {
            if (!mbar_wait(bar_tempty + 8 * acc, ((used >> acc) & 1) ^ 1, abort, budget)) {
              ok = false;
              break;
            }
            tc_fence_after_sync();
            tmem_d = tmem_base + acc * kPairN;
          }
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
            if (k < steps) umma_pair_bf16(tmem_d, dp + k * (kPmn ? 2048 >> 4 : 2), dq + k * (kQmn ? 2048 >> 4 : 2), idesc, !first || k != 0);
          umma_pair_commit(bar_empty + 8 * s);
          if (++s == stages) s = 0, ph ^= 1;
          if (last) {
            umma_pair_commit(bar_tfull + 8 * acc);
            used ^= 1u << acc;
            if (IN_32) acc ^= 1;
          }
        }
        if (!ok) break;
        // (Behind a long sum its accumulator is next again: it is given back once the sum of the parts has been read, too.)
        if (!IN_32 && blocks <= part_blocks) acc ^= 1;
      }
    }
  } else {
    // ---------------- epilogue ----------------
    const int quarter = warp & 3;  // the tensor memory lanes that this warp may read
    const int which = (warp - 2) >> 2;  // of its two warps: takes every other 32 result rows of a tile
    const int et = threadIdx.x - 64;
    const Epilogue& e = a.e;
    uint8_t* stage = turns + (warp - 2) * kTurn;
    // What has no product: rows behind the last group, matrices without rows.  (The first tile's sums are under way meanwhile.)
    const int64_t cta = blockIdx.x, ctas = gridDim.x;
    const int out_cols = kGated ? a.features / 2 : a.features;
    auto clear_row = [&](int64_t row) {
      if (MODE > kForwardGated || a.wide) {
        for (int c = 4 * et; c < out_cols; c += 4 * 32 * kStoreWarps) {
          float v[4] = {0.f, 0.f, 0.f, 0.f};
          if (e.residual != nullptr) load4<1>(e.residual, e.type, row * e.residual_ld + c, 4, v);
          store4<1>(e.out, e.type, row * e.out_ld + c, 4, v);
        }
      } else {
        for (int c = et; c < out_cols; c += 32 * kStoreWarps)
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
    uint32_t acc = 0, used = 0;  // as the matrix instructions' side counts
    const uint32_t lead_tempty = map_to_rank(bar_tempty, 0);
    auto await = [&]() {  // the next accumulator's sums, all of the warp together
      if (!__all_sync(0xffffffffu, mbar_wait(bar_tfull + 8 * acc, (used >> acc) & 1, abort, budget))) return false;
      tc_fence_after_sync();
      return true;
    };
    // The accumulator has been read: tcgen05.wait::ld has returned, and nothing else is handed over.  So the arrival does not release: at
    // cluster scope that waits for the thread's loads and stores under way, some 1500 cycles each time.
    auto release = [&](bool to_other) {  // to_other: the next sum is the other accumulator's
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive_remote_read(lead_tempty + 8 * acc);
      used ^= 1u << acc;
      acc ^= to_other;
    };
    const uint32_t tmem_mine = tmem_base + ((uint32_t)(quarter * 32) << 16);
    int n = 0;           // result rows of the tile that are there
    int64_t row0 = 0;    // the first of them
    auto next = [&](uint32_t i) {
      if (!__all_sync(0xffffffffu, find(i) && !*abort)) return false;
      n = min(cur.n, (MODE == kWeight ? a.result_rows : s_rows[cur.group]) - cur.row0);
      row0 = (MODE == kWeight ? (int64_t)cur.group * a.result_rows : (int64_t)s_start[cur.group]) + cur.row0;
      return true;
    };

    // The next accumulator's sums; before the last part of a long sum those of the parts before are added up beside it.
    bool is_long = false;
    auto await_last = [&]() {
      const int blocks = blocks_of();
      is_long = blocks > a.part_blocks;
      for (int done = 0; done + a.part_blocks < blocks; done += a.part_blocks) {
        if (!await()) return false;
        for (int c = 32 * which; c < n; c += (c & 16) ? 48 : 16) {
          float v[16], before[16];
          __syncwarp();
          tmem_ld_32x16(tmem_mine + acc * kPairN + c, v);
          if (done > 0) tmem_ld_32x16(tmem_mine + (acc ^ 1) * kPairN + c, before);
          tmem_ld_wait();
          if (done > 0) {
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] += before[j];
          }
          tmem_st_32x16(tmem_mine + (acc ^ 1) * kPairN + c, v);
        }
        tmem_st_wait();
        release(false);
      }
      return await();
    };

    // A result in 16 bits: bias, activation and residual on the matrix fragments, turned round by stmatrix, stored by 16 bytes.  The residual
    // comes the same way back.
    auto plain = [&](auto is_bf16) {
      constexpr bool kBf = decltype(is_bf16)::value;
      auto pack = [](float lo, float hi) {
        if constexpr (kBf) {
          const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
          return *reinterpret_cast<const uint32_t*>(&v);
        } else {
          const __half2 v = __floats2half2_rn(lo, hi);
          return *reinterpret_cast<const uint32_t*>(&v);
        }
      };
      auto unpack = [](uint32_t w) {
        if constexpr (kBf) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
        else return __half22float2(*reinterpret_cast<const __half2*>(&w));
      };
      const uint32_t mine = smem_u32(stage);
      constexpr int kRowBytes = kGated ? 32 : 64, kChunks = kRowBytes / 16;  // of a result row, this warp's
      auto chunk_at = [&](int row, int chunk) {  // swizzled: eight rows' chunks lie in different banks
        return row * kRowBytes + ((chunk ^ (kGated ? (row >> 2) & 1 : (row >> 1) & 3)) << 4);
      };
      // What backward needs, in 32 bits, by the same way: the low and the high halves of the values are turned round one after the other, and a
      // lane stores whole sectors.  4096 x 4096 x 1024 with silu and what it keeps: 40.6 us, through `full` 50.6 (nothing kept: 30.4); with
      // swiglu 36.2 by either way.
      auto keep = [&](int c0, const float (&v)[2][16]) {
        auto at64 = [&](int row, int chunk) { return row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4); };
        uint4 half_of[2][4];
#pragma unroll
        for (int high = 0; high < 2; ++high) {
          auto two = [&](float a, float b) { return __byte_perm(__float_as_uint(a), __float_as_uint(b), high ? 0x7632 : 0x5410); };
          __syncwarp();  // the rows before have been read
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float(&f)[16] = v[q >> 1];
            const int h = 2 * (q & 1);
            stmatrix_trans(mine + at64(lane, q), two(f[h], f[h + 1]), two(f[4 + h], f[5 + h]), two(f[8 + h], f[9 + h]), two(f[12 + h], f[13 + h]));
          }
          __syncwarp();
#pragma unroll
          for (int q = 0; q < 4; ++q) half_of[high][q] = *reinterpret_cast<const uint4*>(stage + at64((lane >> 2) + 8 * q, lane & 3));
        }
        const int first = cur.p * kPairM + half * (kGated ? kHalfM / 2 : kHalfM) + quarter * (kGated ? 16 : 32), chunk = lane & 3;
        const int column = first + (kGated ? (chunk & 1) * 8 + (chunk >> 1) * kGateBlock : chunk * 8);
        if (column >= a.features) return;
        float* to = static_cast<float*>(e.pre) + column;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int r = c0 + (lane >> 2) + 8 * q;
          if (r >= n) continue;
          const uint32_t low[4] = {half_of[0][q].x, half_of[0][q].y, half_of[0][q].z, half_of[0][q].w};
          const uint32_t high[4] = {half_of[1][q].x, half_of[1][q].y, half_of[1][q].z, half_of[1][q].w};
          uint32_t w[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) w[j] = __byte_perm(low[j >> 1], high[j >> 1], j & 1 ? 0x7632 : 0x5410);
          st_global_v8(to + (row0 + r) * e.pre_ld, w);
        }
      };
      for (uint32_t i = 0; next(i); ++i) {
        // this thread's features: lane / 4, and 8, 16 (gated: the up row of the first) and 24 behind
        float bias[4] = {0.f, 0.f, 0.f, 0.f};
        const int first = cur.p * kPairM + half * (kGated ? kHalfM / 2 : kHalfM) + quarter * (kGated ? 16 : 32) + (lane >> 2);
        if (MODE <= kForwardGated && e.bias != nullptr) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int c = first + (j & 1) * 8 + (j >> 1) * (kGated ? kGateBlock : 16);
            if (c < e.n) bias[j] = load_as_float(e.bias, e.bias_type, (int64_t)cur.group * e.n + c);
          }
        }
        const int column = (kGated ? cur.p * kHalfM + half * (kHalfM / 2) + quarter * 16 : cur.p * kPairM + half * kHalfM + quarter * 32) + lane % kChunks * 8;
        uint16_t* out = static_cast<uint16_t*>(e.out) + column;
        const bool inside = column < out_cols;
        uint4 carried[kChunks];  // the residual of the step that is next
        auto fetch = [&](int c0) {
          if (MODE > kForwardGated || e.residual == nullptr) return;
          const uint16_t* from = static_cast<const uint16_t*>(e.residual) + (inside ? column : 0);
#pragma unroll
          for (int q = 0; q < kChunks; ++q) {
            const int r = min(c0 + lane / kChunks + q * (32 / kChunks), n - 1);  // (what is not there is not stored)
            carried[q] = *reinterpret_cast<const uint4*>(from + (row0 + r) * e.residual_ld);
          }
        };
        fetch(32 * which);
        if (!await_last()) break;
        for (int c0 = 32 * which; c0 < n; c0 += 64) {
          // fragments: lanes l/4 and l/4 + 8 of a 16-lane half, result rows 8j + 2(l%4) and the next
          uint32_t raw[2][16];
          __syncwarp();
          tmem_ld_16x32(tmem_mine + acc * kPairN + c0, raw[0]);
          tmem_ld_16x32(tmem_mine + (16u << 16) + acc * kPairN + c0, raw[1]);
          tmem_ld_wait();
          if (is_long) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t before[16];
              tmem_ld_16x32(tmem_mine + (h * 16u << 16) + (acc ^ 1) * kPairN + c0, before);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 16; ++j) raw[h][j] = __float_as_uint(__uint_as_float(raw[h][j]) + __uint_as_float(before[j]));
            }
          }
          float v[2][16];
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < 16; ++j) v[h][j] = __uint_as_float(raw[h][j]) + (MODE <= kForwardGated ? bias[2 * h + (j >> 1 & 1)] : 0.f);
          if (MODE > kForwardGated && e.most != nullptr) {
#pragma unroll
            for (int r = 0; r < 8; ++r) {  // (what is not there is not stored)
              const float whole = whole_of(e.most[row0 + min(c0 + 8 * (r >> 1) + 2 * (lane & 3) + (r & 1), n - 1)]);
#pragma unroll
              for (int h = 0; h < 4; ++h) v[h >> 1][4 * (r >> 1) + 2 * (h & 1) + (r & 1)] *= whole;
            }
          }
          if (MODE <= kForwardGated && e.pre != nullptr) keep(c0, v);
          if constexpr (kGated) {
#pragma unroll
            for (int j = 0; j < 16; ++j) v[0][j] = __fmul_rn(__fmul_rn(v[0][j], sigmoid_of(v[0][j])), v[1][j]);
          } else if (MODE == kForward) {
            activate(v[0], e.activation);
            activate(v[1], e.activation);
          }
          __syncwarp();  // the rows before have been read
          if (MODE <= kForwardGated && e.residual != nullptr) {
#pragma unroll
            for (int q = 0; q < kChunks; ++q) *reinterpret_cast<uint4*>(stage + chunk_at(lane / kChunks + q * (32 / kChunks), lane % kChunks)) = carried[q];
            fetch(c0 + 64);
            __syncwarp();
#pragma unroll
            for (int q = 0; q < kChunks; ++q) {
              uint32_t two[4];
              ldmatrix_trans(mine + chunk_at(lane, q), two);
              float(&f)[16] = v[q >> 1];
              const int h = 2 * (q & 1);
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const float2 more = unpack(two[j]);
                f[4 * j + h] += more.x, f[4 * j + h + 1] += more.y;
              }
            }
            __syncwarp();
          }
#pragma unroll
          for (int q = 0; q < kChunks; ++q) {
            const float(&f)[16] = v[q >> 1];
            const int h = 2 * (q & 1);
            stmatrix_trans(mine + chunk_at(lane, q), pack(f[h], f[h + 1]), pack(f[4 + h], f[5 + h]), pack(f[8 + h], f[9 + h]), pack(f[12 + h], f[13 + h]));
          }
          __syncwarp();
#pragma unroll
          for (int q = 0; q < kChunks; ++q) {
            const int r = lane / kChunks + q * (32 / kChunks);
            const uint4 w = *reinterpret_cast<const uint4*>(stage + chunk_at(r, lane % kChunks));
            if (c0 + r < n && inside) *reinterpret_cast<uint4*>(out + (row0 + c0 + r) * e.out_ld) = w;
          }
        }
        release(!is_long);
      }
    };

    // Everything else, in 32 bits through shared memory, 16 result rows at a time; a lane finishes four columns of a row.
    auto full = [&](auto wide) {
      constexpr bool kWide = decltype(wide)::value;
      constexpr int kLanes = kGated ? 4 : 8;                // that share a row of 16 or 32 columns
      constexpr int S = kWide ? 1 : kLanes;
      constexpr int kPer = kLanes / 2;                      // of 16 rows, per lane
      const int f = kWide ? 4 * (lane % kLanes) : lane % kLanes;  // first of its columns, of the warp's
      float* turned = reinterpret_cast<float*>(stage);      // [16 rows][32 lanes of tensor memory]
      for (uint32_t i = 0; next(i); ++i) {
        Columns<S, kGated> mine;
        if constexpr (kGated) {
          mine.out = cur.p * kHalfM + half * (kHalfM / 2) + quarter * 16 + f;
          mine.gate = cur.p * kPairM + half * (kHalfM / 2) + quarter * 16 + f;
          mine.limit = kHalfM;  // whole blocks
        } else {
          mine.out = mine.gate = cur.p * kPairM + half * kHalfM + quarter * 32 + f;
          mine.limit = a.features - mine.out;
        }
        mine.load_bias(e, cur.group);
        auto turn16 = [&](const float (&v)[16]) {
#pragma unroll
          for (int j = 0; j < 16; ++j) turned[j * 32 + lane] = v[j];
        };
        float next_r[kPer][4];  // the residual of the 16 rows that are finished next, under way while these are
        auto fetch = [&](int c0) {
#pragma unroll
          for (int q = 0; q < kPer; ++q) {
            const int at = c0 + lane / kLanes + q * (32 / kLanes);
            if (at < n) mine.load_residual(e, row0 + at, next_r[q]);
          }
        };
        auto after = [&](int c0) { return c0 & 16 ? c0 + 48 : c0 + 16; };  // the warp's 16 rows behind these
        fetch(32 * which);
        auto finish16 = [&](int c0, auto&& turn) {  // result rows c0 .. c0 + 15 of the tile
          float r[kPer][4];
#pragma unroll
          for (int q = 0; q < kPer; ++q)
#pragma unroll
            for (int j = 0; j < 4; ++j) r[q][j] = next_r[q][j];
          fetch(after(c0));
          __syncwarp();  // the rows before have been read
          turn();
          __syncwarp();
#pragma unroll
          for (int q = 0; q < kPer; ++q) {
            const int in_turn = lane / kLanes + q * (32 / kLanes), at = c0 + in_turn;
            if (at >= n) continue;
            const float* from = turned + in_turn * 32 + f;
            float z[4], up[4];
            // gated: 16 gate rows and their 16 up rows
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              z[j] = from[j * S];
              up[j] = kGated ? from[16 + j * S] : 0.f;
            }
            mine.finish(e, row0 + at, z, up, r[q]);
          }
        };
        if constexpr (IN_32) {
          constexpr int kBlocks = kSumRows / 64;
          float sum[kBlocks][2][16];  // this warp's 32 result rows of every 64
          const int parts = (a.k_blocks + kSumBlocks - 1) / kSumBlocks;
          bool ok = true;
          for (int p = 0; p < parts; ++p) {
            if (!(ok = await())) break;
#pragma unroll
            for (int c = 0; c < kBlocks; ++c) {
              if (32 * which + 64 * c >= n) continue;
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                float v[16];
                __syncwarp();
                tmem_ld_32x16(tmem_mine + acc * kPairN + 32 * which + 64 * c + 16 * h, v);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 16; ++j) sum[c][h][j] = p == 0 ? v[j] : sum[c][h][j] + v[j];
              }
            }
            release(true);
          }
          if (!ok) break;
#pragma unroll 1
          for (int b = 0; b < 2 * kBlocks; ++b) {  // one copy of the code behind
            const int c0 = 32 * which + 64 * (b >> 1) + 16 * (b & 1);
            if (c0 >= n) break;
            finish16(c0, [&] {
#pragma unroll
              for (int of = 0; of < 2 * kBlocks; ++of)
                if (of == b) turn16(sum[of >> 1][of & 1]);
            });
          }
        } else {
          if (!await_last()) break;
          for (int c0 = 32 * which; c0 < n; c0 += 64)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if (c0 + 16 * h >= n) continue;
              float v[16];
              __syncwarp();
              tmem_ld_32x16(tmem_mine + acc * kPairN + c0 + 16 * h, v);
              tmem_ld_wait();
              if (is_long) {
                float before[16];
                tmem_ld_32x16(tmem_mine + (acc ^ 1) * kPairN + c0 + 16 * h, before);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 16; ++j) v[j] += before[j];
              }
              finish16(c0 + 16 * h, [&] { turn16(v); });
            }
          release(!is_long);
        }
      }
    };
    // (The gradients' rows are always of whole words on boundaries.)
    if (!IN_32 && (MODE > kForwardGated || a.plain)) {
      if (e.type == Type::kBf16) plain(std::true_type{});
      else plain(std::false_type{});
    } else if constexpr (MODE <= kForwardGated) {
      if (a.wide) full(std::true_type{});
      else full(std::false_type{});
    }
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

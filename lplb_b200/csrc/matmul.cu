// Launchers of the product with an epilogue and of its gradients, and the kernel that takes a gradient through the activation.
#include "matmul_api.h"

#include <atomic>

#include "matmul.cuh"
#include "matmul_cost.h"
#include "matmul_few.cuh"
#include "tensor_map.h"

namespace lplb {
namespace ops {

namespace {

// ---- the activation's gradient -----------------------------------------------------------------------
// dz = dout * act'(z), rounded to the operands' type for the products behind it, and the sum of dz (before the rounding) over
// parts of a group's rows.  A CTA has 256 columns of z, a part of a group's rows, eight of them at a time; bound by DRAM.
// 8192 x 4096 in bf16 through silu with the bias's gradient: 49 us, 5.5 TB/s (one row at a time for each warp 53, four 60, two converted
// as they come 56); 16384 x 4096 of 32 experts through swiglu 80 us, 5.8 TB/s; gelu of 32-bit results 61, by its instructions.
constexpr int kPreColumns = 256, kPreRows = 8;

// (which activation is asked once, not for each value)
__device__ __forceinline__ void through(float (&d)[2][4], const float (&z)[2][4], int activation) {
  if (activation == kSilu) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float u = z[i / 4][i % 4], s = sigmoid_of(u);
      d[i / 4][i % 4] *= s * (1.f + u * (1.f - s));
    }
  } else if (activation == kGelu) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float u = z[i / 4][i % 4];
      float bell;
      const float cdf = normal_cdf(u, bell);
      d[i / 4][i % 4] *= cdf + u * 0.3989422804f * bell;  // 1 / sqrt(2 pi)
    }
  } else if (activation == kRelu) {
#pragma unroll
    for (int i = 0; i < 8; ++i) d[i / 4][i % 4] = z[i / 4][i % 4] > 0.f ? d[i / 4][i % 4] : 0.f;
  }
}

struct PreArgs {
  const void* dout;
  const void* pre;
  const int* rows;
  void* dz;
  void* dz_weight;
  uint32_t* row_most;
  uint32_t* column_most;
  void* dbias;   // where one part is all of a group
  float* parts;  // [groups, splits, n]
  int64_t dout_ld, pre_ld, dz_ld;
  int m, n, groups, splits, activation;
  Type type, out_type, bias_type;
};

// dz in parts of a power of two takes two passes: the largest magnitudes (and the bias's gradient), then dz.  The magnitudes go to memory by
// atomicMax, whose order changes nothing.  1001 x 4100 x 2064 in float16 through gelu, all gradients, captured: 117 us, by one pass, which
// loses what float16 does not hold, 102; cleared by two memsets instead of a kernel 123.
enum Pass : int { kOnePass = 0, kMost = 1, kParts = 2 };

// VEC: everything is there in whole vectors of four values
template <bool VEC, bool GATED, Pass PASS>
__global__ void __launch_bounds__(256) pre_gradient_kernel(const PreArgs a) {
  constexpr int S = VEC ? 1 : GATED ? 32 : 64;          // the thread's columns are this far apart
  constexpr int kVectors = GATED ? 1 : 2;               // of four columns: 32 lanes x 4 (and 128 behind, or the up columns)
  constexpr int kNext = VEC ? 128 : 32;                 // from the thread's first vector to its second
  __shared__ float s_sum[kPreRows][kPreColumns];
  __shared__ long long s_before[8];
  wait_predecessors();
  allow_successor();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int split = blockIdx.y, group = blockIdx.z;
  int from = 0, rows = a.m;
  if (a.rows != nullptr) {  // the group's rows, none beyond the last
    long long before = 0;
    for (int e = threadIdx.x; e < group; e += 256) before += max(a.rows[e], 0);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
    if (lane == 0) s_before[warp] = before;
    __syncthreads();
    before = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) before += s_before[w];
    from = (int)min((long long)a.m, before);
    rows = (int)min((long long)a.m - from, (long long)max(a.rows[group], 0));
  }
  const int r0 = from + (int)((int64_t)rows * split / a.splits), r1 = from + (int)((int64_t)rows * (split + 1) / a.splits);
  // the first column of a vector in dout, and in z
  int at_out[kVectors], at_z[kVectors], limit[kVectors];
#pragma unroll
  for (int v = 0; v < kVectors; ++v) {
    const int f = (VEC ? 4 * lane : lane) + v * kNext;
    at_out[v] = GATED ? blockIdx.x * kGateBlock + f : blockIdx.x * kPreColumns + f;
    at_z[v] = blockIdx.x * kPreColumns + f;
    limit[v] = GATED ? 4 * S : a.n - at_z[v];
  }
  float sum[2][4] = {};
  uint32_t most[2][4] = {};   // kMost
  float part[2][4];           // kParts: of the thread's columns
  if constexpr (PASS == kParts) {
#pragma unroll
    for (int v = 0; v < 2; ++v)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool there = GATED || limit[v % kVectors] > (VEC ? 0 : j * S);
        const int column = at_z[GATED ? 0 : v % kVectors] + (GATED && v ? kGateBlock : 0) + j * S;
        part[v][j] = there && a.column_most != nullptr ? part_of(a.column_most[(int64_t)group * a.n + column]) : 1.f;
      }
  }
  constexpr int kAtOnce = VEC ? 2 : 1;  // rows whose loads are under way together
  for (int base = r0 + warp; base < r1; base += kPreRows * kAtOnce) {
    float d[kAtOnce][2][4] = {}, z[kAtOnce][2][4] = {};
    uint4 raw[kAtOnce][kVectors] = {};
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int64_t r = min(base + i * kPreRows, r1 - 1);  // (the last row again, and left out below)
#pragma unroll
      for (int v = 0; v < kVectors; ++v) {
        if constexpr (VEC) {  // (as they stand: turned into 32 bits here, a row would wait for the one before)
          if (limit[v] > 0) {
            const int64_t at = r * a.dout_ld + at_out[v];
            if (a.out_type == Type::kF32) {
              raw[i][v] = *reinterpret_cast<const uint4*>(static_cast<const float*>(a.dout) + at);
            } else {
              const uint2 two = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(a.dout) + at);
              raw[i][v].x = two.x, raw[i][v].y = two.y;
            }
          }
        } else {
          load4<S>(a.dout, a.out_type, r * a.dout_ld + at_out[v], limit[v], d[i][v]);
        }
        if (a.pre != nullptr) load4<S>(a.pre, Type::kF32, r * a.pre_ld + at_z[v], limit[v], z[i][v]);
      }
      if (GATED) load4<S>(a.pre, Type::kF32, r * a.pre_ld + at_z[0] + kGateBlock, limit[0], z[i][1]);
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int64_t r = base + i * kPreRows;
      if (r >= r1) break;
      if constexpr (VEC) {
#pragma unroll
        for (int v = 0; v < kVectors; ++v) {
          const uint32_t w[4] = {raw[i][v].x, raw[i][v].y, raw[i][v].z, raw[i][v].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (a.out_type == Type::kF32) d[i][v][j] = __uint_as_float(w[j]);
            else if (a.out_type == Type::kBf16) d[i][v][j] = __uint_as_float(j & 1 ? w[j / 2] & 0xFFFF0000u : w[j / 2] << 16);
            else d[i][v][j] = __half2float(__ushort_as_half((unsigned short)(w[j / 2] >> (16 * (j & 1)))));
          }
        }
      }
      if (GATED) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float s = sigmoid_of(z[i][0][j]), g = d[i][0][j];
          d[i][0][j] = g * z[i][1][j] * s * (1.f + z[i][0][j] * (1.f - s));
          d[i][1][j] = g * z[i][0][j] * s;
        }
      } else {
        through(d[i], z[i], a.activation);
      }
      if constexpr (PASS == kMost) {
        uint32_t of_row = 0;
#pragma unroll
        for (int v = 0; v < 2; ++v)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t magnitude = finite_magnitude(d[i][v][j]);
            most[v][j] = max(most[v][j], magnitude);
            of_row = max(of_row, magnitude);
          }
        if (a.row_most != nullptr) {
          of_row = __reduce_max_sync(0xffffffffu, of_row);
          if (lane == 0) atomicMax(a.row_most + r, of_row);
        }
      }
      const float of_row = PASS == kParts && a.row_most != nullptr ? part_of(a.row_most[r]) : 1.f;
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        const int w = GATED ? 0 : v;
        const int64_t at = r * a.dz_ld + at_z[w] + (GATED && v ? kGateBlock : 0);
        if (PASS != kMost && a.dz != nullptr) {
          float whole_row[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) whole_row[j] = PASS == kParts ? d[i][v][j] * of_row : d[i][v][j];
          store4<S>(a.dz, a.type, at, limit[w], whole_row);
        }
        if (PASS == kParts && a.dz_weight != nullptr) {
          float by_column[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) by_column[j] = d[i][v][j] * part[v][j];
          store4<S>(a.dz_weight, a.type, at, limit[w], by_column);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[v][j] += d[i][v][j];
      }
    }
  }
  if constexpr (PASS == kMost) {
    if (a.column_most != nullptr) {
      uint32_t(&s_most)[kPreRows][kPreColumns] = *reinterpret_cast<uint32_t(*)[kPreRows][kPreColumns]>(&s_sum);
#pragma unroll
      for (int v = 0; v < 2; ++v)
#pragma unroll
        for (int j = 0; j < 4; ++j) s_most[warp][(VEC ? 4 * lane : lane) + j * S + (GATED ? v * kGateBlock : v * kNext)] = most[v][j];
      __syncthreads();
      const int column = blockIdx.x * kPreColumns + threadIdx.x;
      uint32_t all = 0;
#pragma unroll
      for (int w = 0; w < kPreRows; ++w) all = max(all, s_most[w][threadIdx.x]);
      if (column < a.n && all != 0) atomicMax(a.column_most + (int64_t)group * a.n + column, all);
      __syncthreads();  // the sums come to the same place
    }
  }
  if (a.dbias == nullptr && a.parts == nullptr) return;
#pragma unroll
  for (int v = 0; v < 2; ++v)
#pragma unroll
    for (int j = 0; j < 4; ++j) s_sum[warp][(VEC ? 4 * lane : lane) + j * S + (GATED ? v * kGateBlock : v * kNext)] = sum[v][j];
  __syncthreads();
  const int column = blockIdx.x * kPreColumns + threadIdx.x;
  if (column >= a.n) return;
  float all = 0.f;
#pragma unroll
  for (int w = 0; w < kPreRows; ++w) all += s_sum[w][threadIdx.x];
  if (a.parts != nullptr)
    a.parts[((int64_t)group * a.splits + split) * a.n + column] = all;
  else
    store_float(a.dbias, a.bias_type, (int64_t)group * a.n + column, all);
}

// The magnitudes before the first pass.
__global__ void __launch_bounds__(256) clear_most_kernel(uint32_t* rows, int64_t n_rows, uint32_t* columns, int64_t n_columns) {
  wait_predecessors();
  allow_successor();
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < n_rows) rows[i] = 0;
  if (i < n_columns) columns[i] = 0;
}

// dbias[g, c] = sum of its parts, in their order
__global__ void __launch_bounds__(256) bias_parts_kernel(const float* parts, void* dbias, Type type, int64_t n, int splits, int64_t total) {
  wait_predecessors();
  allow_successor();
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= total) return;
  const int64_t group = i / n, column = i - group * n;
  const float* from = parts + group * splits * n + column;
  float all = 0.f;
  for (int s0 = 0; s0 < splits; s0 += 16) {  // 16 loads under way
    float v[16];
#pragma unroll
    for (int s = 0; s < 16; ++s) v[s] = from[min(s0 + s, splits - 1) * n];
#pragma unroll
    for (int s = 0; s < 16; ++s) all += s0 + s < splits ? v[s] : 0.f;
  }
  store_float(dbias, type, i, all);
}

uint64_t address(const void* p) { return reinterpret_cast<uintptr_t>(p); }
// Whether four neighbouring values of rows `ld` apart always start on a boundary of their size.
bool fours(const void* p, int64_t ld, Type type) { return p == nullptr || (ld % 4 == 0 && address(p) % (type == Type::kF32 ? 16 : 8) == 0); }

// ---- tensor maps ----------------------------------------------------------------------------------------
constexpr CUtensorMapDataType kMapType = CU_TENSOR_MAP_DATA_TYPE_UINT16;  // TMA copies bits; the zeros it fills in are those of both types

// [rows, cols] with rows `ld` apart, boxes of 64 columns
cudaError_t map_2d(CUtensorMap* map, const void* base, uint64_t rows, uint64_t cols, uint64_t ld, uint32_t box_rows) {
  const cuuint64_t dims[2] = {cols, rows}, strides[1] = {ld * 2};
  const cuuint32_t box[2] = {(cuuint32_t)kPairK, box_rows};
  return encode_tensor_map(map, kMapType, base, 2, dims, strides, box) == 0 ? cudaSuccess : cudaErrorInvalidValue;
}
// [matrices, rows, cols]: zeros behind a matrix's last row, not the next one's values
cudaError_t map_3d(CUtensorMap* map, const void* base, uint64_t matrices, uint64_t rows, uint64_t cols, uint32_t box_rows) {
  const cuuint64_t dims[3] = {cols, rows, matrices}, strides[2] = {cols * 2, rows * cols * 2};
  const cuuint32_t box[3] = {(cuuint32_t)kPairK, box_rows, 1};
  return encode_tensor_map(map, kMapType, base, 3, dims, strides, box) == 0 ? cudaSuccess : cudaErrorInvalidValue;
}
// MN-major operands whose columns come in whole chunks of 64: [rows, cols] as [chunks, rows, 64], boxes of two chunks
cudaError_t map_chunks(CUtensorMap* map, const void* base, uint64_t rows, uint64_t cols, uint64_t ld, uint32_t box_rows) {
  const cuuint64_t dims[3] = {kChunk, rows, cols / kChunk}, strides[2] = {ld * 2, kChunk * 2};
  const cuuint32_t box[3] = {kChunk, box_rows, 2};
  return encode_tensor_map(map, kMapType, base, 3, dims, strides, box) == 0 ? cudaSuccess : cudaErrorInvalidValue;
}
cudaError_t map_chunks(CUtensorMap* map, const void* base, uint64_t matrices, uint64_t rows, uint64_t cols) {
  const cuuint64_t dims[4] = {kChunk, rows, cols / kChunk, matrices}, strides[3] = {cols * 2, kChunk * 2, rows * cols * 2};
  const cuuint32_t box[4] = {kChunk, kPairK, 2, 1};
  return encode_tensor_map(map, kMapType, base, 4, dims, strides, box) == 0 ? cudaSuccess : cudaErrorInvalidValue;
}
// Weights in blocks of 128 gate rows and their 128 up rows, dealt out so that 32 rows in shared memory are 16 gate rows and their
// 16 up rows.
cudaError_t map_gated(CUtensorMap* map, const void* base, uint64_t rows, uint64_t cols) {
  const cuuint64_t row = cols * 2;
  const cuuint64_t dims[5] = {cols, 16, 2, kGateBlock / 16, rows / (2 * kGateBlock)};
  const cuuint64_t strides[4] = {row, kGateBlock * row, 16 * row, 2 * kGateBlock * row};
  const cuuint32_t box[5] = {(cuuint32_t)kPairK, 16, 2, kHalfM / 32, 1};
  return encode_tensor_map(map, kMapType, base, 5, dims, strides, box) == 0 ? cudaSuccess : cudaErrorInvalidValue;
}
cudaError_t maps_of_rows(PairMaps* maps, const void* base, uint64_t rows, uint64_t cols, uint64_t ld) {
  cudaError_t err = cudaSuccess;
  for (int b = 0; b < 4 && err == cudaSuccess; ++b) err = map_2d(&maps->q[b], base, rows, cols, ld, kPairN / 2 >> b);
  return err;
}

// ---- CTA pairs --------------------------------------------------------------------------------------------
// Of a weight's gradient: the groups' rows are what is summed, here as if they were equal.
int weight_steps(int64_t result_rows, int64_t rows, int groups, int64_t tiles_p, int n_sm) {
  return pair_cost(result_rows, kWeightStep, kPairN, tiles_p * groups, (rows / groups + kPairK - 1) / kPairK, n_sm).steps;
}

template <Mode MODE, bool IN_32 = false>
cudaError_t launch_pairs(const PairMaps& maps, PairArgs& a, int device, cudaStream_t stream) {
  auto kernel = pair_matmul_kernel<MODE, IN_32>;
  static std::atomic<bool> prepared[kMaxDevices];
  int n_sm = 0;
  cudaError_t err = multiprocessors(device, &n_sm);
  if (err != cudaSuccess) return err;
  if (!prepared[device].load(std::memory_order_relaxed)) {
    err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kPairSmem);
    if (err != cudaSuccess) return err;
    prepared[device].store(true, std::memory_order_relaxed);
  }
  if ((err = ops_error_word(device, &a.status)) != cudaSuccess) return err;
  a.budget_ns = wait_budget_ns();
  a.part_blocks = longest_part(a.e.type) / kPairK;
  if (a.p_chunks == 0) a.p_chunks = 1;
  if (a.q_chunks == 0) a.q_chunks = 1;
  a.tiles_p = (a.features + kPairM - 1) / kPairM;
  const int out_cols = MODE == kForwardGated ? a.features / 2 : a.features;
  a.plain = a.e.type != Type::kF32 && a.e.residual_ld % 8 == 0 && address(a.e.residual) % 16 == 0 && address(a.e.pre) % 32 == 0 && a.e.pre_ld % 8 == 0 && out_cols % 8 == 0 && a.e.out_ld % 8 == 0 && address(a.e.out) % 16 == 0;
  if (MODE > kForwardGated && !(a.wide && a.plain)) return cudaErrorMisalignedAddress;
  const int most_rows = IN_32 ? kSumRows : kPairN;
  a.tile_steps = most_rows / PairTile<MODE>::kStep;
  if (MODE == kWeight) a.tile_steps = weight_steps(a.result_rows, a.n_rows, a.groups, a.tiles_p, n_sm);
  else if (a.rows == nullptr) a.tile_steps = pair_cost(a.n_rows, PairTile<MODE>::kStep, most_rows, a.tiles_p, a.k_blocks, n_sm).steps;
  return launch_after(kernel, dim3(n_sm & ~1), dim3(kPairThreads), kPairSmem, stream, maps, a);
}

Epilogue epilogue_of(const Matmul& p) {
  Epilogue e{};
  e.bias = p.bias;
  e.residual = p.residual;
  e.out = p.out;
  e.pre = p.pre;
  e.residual_ld = p.residual_ld;
  e.out_ld = p.out_ld;
  e.pre_ld = p.pre_ld;
  e.n = (int)p.n;
  e.activation = p.activation;
  e.type = p.out_type;
  e.bias_type = p.bias_type;
  return e;
}
int is_wide(const Matmul& p) {
  return p.n % 4 == 0 && fours(p.out, p.out_ld, p.out_type) && fours(p.residual, p.residual_ld, p.out_type) && fours(p.pre, p.pre_ld, Type::kF32) &&
         fours(p.bias, p.n, p.bias_type);
}

// A result in 32 bits whose sum is longer than one part.  us, sums of one part in tiles of up to 256 rows and in registers: 600 x 4096 x 512 9.7,
// 13.1; 8192 x 1000 x 512 18.0, 24.2.
bool sums_in_parts(const Matmul& p) { return p.out_type == Type::kF32 && p.k > longest_part(p.out_type); }

cudaError_t launch_forward(const Matmul& p, int device, cudaStream_t stream) {
  PairMaps maps{};
  PairArgs a{};
  a.rows = p.rows;
  a.groups = p.rows ? p.groups : 1;
  a.n_rows = (int)p.m;
  a.features = (int)p.n;
  a.k_blocks = (int)((p.k + kPairK - 1) / kPairK);
  a.wide = is_wide(p);
  a.idesc = sm100::umma_idesc_16(p.type == Type::kBf16, false, false);
  a.e = epilogue_of(p);
  cudaError_t err = maps_of_rows(&maps, p.a, p.m, p.k, p.a_ld);
  if (err != cudaSuccess) return err;
  const bool in_parts = sums_in_parts(p);
  if (p.activation == kSwiglu) {
    if ((err = map_gated(&maps.p[0], p.b, (uint64_t)a.groups * p.n, p.k)) != cudaSuccess) return err;
    return in_parts ? launch_pairs<kForwardGated, true>(maps, a, device, stream) : launch_pairs<kForwardGated>(maps, a, device, stream);
  }
  if ((err = map_3d(&maps.p[0], p.b, a.groups, p.n, p.k, kHalfM)) != cudaSuccess) return err;
  return in_parts ? launch_pairs<kForward, true>(maps, a, device, stream) : launch_pairs<kForward>(maps, a, device, stream);
}

// ---- few rows -----------------------------------------------------------------------------------------------
// us, cold weights, rings of 96 KB, for which the next kernel's CTAs could be set up beside these, and of 192: 64 x 4096 x 7168 16.3,
// 13.8; 128 x 4096 x 7168 19.8, 16.0; 16 x 4096 x 4096 9.8, 9.3.
constexpr uint32_t kFewRing = 192 * 1024;
constexpr int kFewSmem = 226 * 1024;  // at most

template <typename Kernel>
cudaLaunchConfig_t few_config(cudaLaunchAttribute (&attrs)[2], int ctas, int split, uint32_t smem, cudaStream_t stream, Kernel) {
  attrs[0].id = cudaLaunchAttributeClusterDimension;
  attrs[0].val.clusterDim.x = split;
  attrs[0].val.clusterDim.y = attrs[0].val.clusterDim.z = 1;
  attrs[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(ctas);
  config.blockDim = dim3(kFewBlock);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  config.attrs = attrs;
  config.numAttrs = 2;
  return config;
}
// Clusters of `split` CTAs that the device holds at once, one CTA per SM.
template <typename Kernel>
cudaError_t resident_clusters(int device, int split, Kernel kernel, int* clusters) {
  static std::atomic<int> known[kMaxDevices][kFewMostSplit + 1];
  *clusters = known[device][split].load(std::memory_order_relaxed);
  if (*clusters > 0) return cudaSuccess;
  cudaLaunchAttribute attrs[2]{};
  cudaLaunchConfig_t config = few_config(attrs, split, split, kFewSmem, nullptr, kernel);
  config.numAttrs = 1;
  const cudaError_t err = cudaOccupancyMaxActiveClusters(clusters, kernel, &config);
  if (err == cudaSuccess) known[device][split].store(*clusters, std::memory_order_relaxed);
  return err;
}
// Accumulators, and stages of the ring, of CTAs with `cols` rows of a and `blocks` k blocks, at most `part` of them to an accumulator.
int few_chains(int cols, int blocks, int part) {
  int chains = 1;
  while (chains * part < blocks && (chains + 1) * cols <= kFewMostRows) ++chains;
  return chains;
}
int few_stages(int cols, int blocks) {
  const int stages = (int)(kFewRing / (kFewWeightStage + cols * kFewKBytes));
  return stages < kFewStageMax ? stages < blocks ? stages : blocks : kFewStageMax < blocks ? kFewStageMax : blocks;
}

// How many CTAs share a tile's k blocks, and how many rows of a a CTA has: so that the cycles of block_cycles' kind are least.  cols is 0
// where nothing fits.
struct FewCost {
  int64_t cycles;
  int split, cols;
};
cudaError_t prepare_few(int device) {
  static std::atomic<bool> prepared[kMaxDevices];
  if (prepared[device].load(std::memory_order_relaxed)) return cudaSuccess;
  cudaError_t err = cudaFuncSetAttribute(few_product_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewSmem);
  if (err == cudaSuccess) err = cudaFuncSetAttribute(few_product_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewSmem);
  if (err == cudaSuccess) prepared[device].store(true, std::memory_order_relaxed);
  return err;
}
cudaError_t few_cost(const Matmul& p, int device, FewCost* best) {
  cudaError_t err = prepare_few(device);
  if (err != cudaSuccess) return err;
  const bool in_32 = p.out_type == Type::kF32;
  const int most_rows = in_32 ? kFewMostRows / 2 : kFewMostRows;  // two accumulators at least
  // (32 bits and up to eight parts of the rows: the search is one of the call's five microseconds at most)
  const int m = (int)p.m, tiles = (int)((p.n + kFewTileRows - 1) / kFewTileRows), k_blocks = (int)((p.k + kPairK - 1) / kPairK);
  const int part = longest_part(p.out_type) / kPairK;
  *best = {INT64_MAX, 0, 0};
  for (int s = 1; s <= kFewMostSplit && s <= k_blocks; ++s) {
    int fit = 0;
    if ((err = resident_clusters(device, s, few_product_kernel<false>, &fit)) != cudaSuccess) return err;
    if (fit < 1) continue;
    const int blocks = (k_blocks + s - 1) / s, least_groups = (m + most_rows - 1) / most_rows;
    for (int g = least_groups; g <= (m + 15) / 16 && g < least_groups + 8; ++g) {
      const int cols = ((m + g - 1) / g + 15) / 16 * 16, groups = (m + cols - 1) / cols;
      if ((int64_t)few_chains(cols, blocks, part) * part < blocks) continue;  // its parts would be longer than the pairs'
      const int64_t cycles = few_cycles((int64_t)tiles * groups, fit, blocks, cols, s);
      if (cycles < best->cycles) *best = {cycles, s, cols};
    }
  }
  return cudaSuccess;
}

template <bool GATED>
cudaError_t launch_few(const Matmul& p, const FewCost& how, int device, cudaStream_t stream) {
  auto kernel = few_product_kernel<GATED>;
  FewProductArgs a{};
  cudaError_t err = ops_error_word(device, &a.status);
  if (err != cudaSuccess) return err;
  a.budget_ns = wait_budget_ns();
  a.m = (int)p.m;
  a.k_blocks = (int)((p.k + kPairK - 1) / kPairK);
  a.wide = is_wide(p);
  a.idesc = sm100::umma_idesc_16(p.type == Type::kBf16, false, false);
  a.e = epilogue_of(p);
  a.tiles = (int)((p.n + kFewTileRows - 1) / kFewTileRows);
  a.cols = how.cols;
  const int split = how.split, groups = (a.m + a.cols - 1) / a.cols, blocks = (a.k_blocks + split - 1) / split;
  a.stages = few_stages(a.cols, blocks);
  a.chains = few_chains(a.cols, blocks, longest_part(p.out_type) / kPairK);
  CUtensorMap map_b, map_a;
  if ((err = map_2d(&map_b, p.b, p.n, p.k, p.k, GATED ? kFewTileRows / 2 : kFewTileRows)) != cudaSuccess) return err;
  if ((err = map_2d(&map_a, p.a, p.m, p.k, p.a_ld, a.cols)) != cudaSuccess) return err;
  cudaLaunchAttribute attrs[2]{};
  const cudaLaunchConfig_t config = few_config(attrs, a.tiles * groups * split, split, FewProductLayout(a.cols, a.chains, a.stages).request, stream, kernel);
  return cudaLaunchKernelEx(&config, kernel, map_b, map_a, a);
}

bool refused(int64_t m, int64_t n, int64_t k, int groups, int device) {
  return m < 0 || n < 1 || k < 1 || groups < 1 || groups > kMatmulMaxGroups || m > kMaxRows || n > kMaxRows || k > kMaxRows || device < 0 ||
         device >= kMaxDevices;
}

// ---- a weight's gradient over groups: their last blocks ------------------------------------------------------
// Rows of a and dz behind a group's last whole block of 64, and zeros up to a multiple of 16 (the rest is not read).  By words of
// 16 bytes; a row's last one may end behind its values, with zeros.
struct LastBlocks {
  const void* from[2];
  void* to[2];
  int64_t from_ld[2], to_ld[2], bytes[2];  // in bytes
  int words[2];
  const int* rows;
  int groups, m;
};
__global__ void __launch_bounds__(256) last_blocks_kernel(const LastBlocks a) {
  __shared__ long long s_before[8];
  wait_predecessors();
  allow_successor();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, group = blockIdx.y;
  long long before = 0;
  for (int e = threadIdx.x; e < group; e += 256) before += max(a.rows[e], 0);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
  if (lane == 0) s_before[warp] = before;
  __syncthreads();
  before = 0;
#pragma unroll
  for (int w = 0; w < 8; ++w) before += s_before[w];
  const int first = (int)min((long long)a.m, before), rows = (int)min((long long)a.m - first, (long long)max(a.rows[group], 0));
  const int count = rows % kPairK, padded = (count + 15) / 16 * 16;
  int word = blockIdx.x * 256 + threadIdx.x;
  const int which = word >= a.words[0];
  if (which) word -= a.words[0];
  if (word >= a.words[which]) return;
  const uint8_t* from = static_cast<const uint8_t*>(a.from[which]) + (int64_t)(first + rows - count) * a.from_ld[which] + (int64_t)word * 16;
  uint8_t* to = static_cast<uint8_t*>(a.to[which]) + (int64_t)group * kPairK * a.to_ld[which] + (int64_t)word * 16;
  const int64_t left = a.bytes[which] - (int64_t)word * 16;
  constexpr int kAtOnce = 8;  // rows; nothing is asked between their loads
  for (int r0 = blockIdx.z * kAtOnce; r0 < padded; r0 += gridDim.z * kAtOnce) {
    uint4 v[kAtOnce];
    if (left >= 16) {
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) v[i] = ld_behind_wait(reinterpret_cast<const uint4*>(from + min(r0 + i, count - 1) * a.from_ld[which]));
    } else {  // nothing behind the row's values is read
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        alignas(16) uint16_t part[8] = {};
        for (int c = 0; c < left / 2; ++c) part[c] = reinterpret_cast<const uint16_t*>(from + min(r0 + i, count - 1) * a.from_ld[which])[c];
        v[i] = *reinterpret_cast<const uint4*>(part);
      }
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      if (r0 + i >= count) v[i] = make_uint4(0, 0, 0, 0);
      if (r0 + i < padded) *reinterpret_cast<uint4*>(to + (r0 + i) * a.to_ld[which]) = v[i];
    }
  }
}
struct WeightCopies {
  int64_t a_ld, dz_ld, a_bytes, bytes;  // values; bytes of a's copies, and of all
};
WeightCopies weight_copies(const MatmulWeight& p) {
  WeightCopies c;
  c.a_ld = (p.k + 7) / 8 * 8;
  c.dz_ld = (p.n + 7) / 8 * 8;
  c.a_bytes = (int64_t)p.groups * kPairK * c.a_ld * 2;
  c.bytes = c.a_bytes + (int64_t)p.groups * kPairK * c.dz_ld * 2;
  return c;
}

PreArgs pre_args(const MatmulPre& p) {
  PreArgs a{};
  a.dout = p.dout;
  a.pre = p.pre;
  a.rows = p.rows;
  a.dz = p.dz;
  a.dz_weight = p.dz_weight;
  a.row_most = p.row_most;
  a.column_most = p.column_most;
  a.dbias = p.dbias;
  a.parts = p.parts;
  a.dout_ld = p.dout_ld;
  a.pre_ld = p.pre_ld;
  a.dz_ld = p.dz_ld;
  a.m = (int)p.m;
  a.n = (int)p.n;
  a.groups = p.rows ? p.groups : 1;
  a.activation = p.activation;
  a.type = p.type;
  a.out_type = p.out_type;
  a.bias_type = p.bias_type;
  return a;
}

}  // namespace

cudaError_t launch_matmul(const Matmul& p, int device, cudaStream_t stream) {
  if (refused(p.m, p.n, p.k, p.groups, device) || p.k % 8 || (p.activation == kSwiglu && p.n % (2 * kGateBlock))) return cudaErrorInvalidValue;
  if (p.m == 0) return cudaSuccess;
  // One matrix and not too many rows: by the kernel that takes the fewer cycles.  us, few_product_kernel and the pairs, cold weights: 64 x
  // 4096 x 7168 13.8, 20.5; 128 x 2048 x 2048 7.3, 8.9; 400 x 1000 x 4096 10.0, 13.0; 200 x 7168 x 2048 14.0, 11.2; 600 x 4096 x 1024 13.6, 8.9.
  if (p.rows == nullptr && p.m <= 2048) {
    int n_sm = 0;
    FewCost few{};
    cudaError_t err = multiprocessors(device, &n_sm);
    if (err == cudaSuccess) err = few_cost(p, device, &few);
    if (err != cudaSuccess) return err;
    const PairCost pairs = pair_cost(p.m, kRowStep, sums_in_parts(p) ? kSumRows : kPairN, (p.n + kPairM - 1) / kPairM, (p.k + kPairK - 1) / kPairK, n_sm);
    if (few.cols > 0 && few.cycles <= pairs.cycles) return p.activation == kSwiglu ? launch_few<true>(p, few, device, stream) : launch_few<false>(p, few, device, stream);
  }
  return launch_forward(p, device, stream);
}

cudaError_t launch_matmul_input(const MatmulInput& p, int device, cudaStream_t stream) {
  if (refused(p.m, p.n, p.k, p.groups, device) || p.k % 8 || p.dz_ld % 8) return cudaErrorInvalidValue;
  if (p.m == 0) return cudaSuccess;
  PairMaps maps{};
  PairArgs a{};
  a.rows = p.rows;
  a.groups = p.rows ? p.groups : 1;
  a.n_rows = (int)p.m;
  a.features = (int)p.k;
  a.k_blocks = (int)((p.n + kPairK - 1) / kPairK);
  a.wide = fours(p.da, p.da_ld, p.type);
  a.idesc = sm100::umma_idesc_16(p.type == Type::kBf16, true, false);
  a.e.out = p.da;
  a.e.most = p.most;
  a.e.out_ld = p.da_ld;
  a.e.n = (int)p.k;
  a.e.type = p.type;
  cudaError_t err = maps_of_rows(&maps, p.dz, p.m, p.n, p.dz_ld);
  a.p_chunks = p.k % kChunk == 0 && p.k > kChunk ? 2 : 1;
  if (err == cudaSuccess) err = a.p_chunks == 2 ? map_chunks(&maps.p[0], p.b, a.groups, p.n, p.k) : map_3d(&maps.p[0], p.b, a.groups, p.n, p.k, kPairK);
  return err != cudaSuccess ? err : launch_pairs<kInput>(maps, a, device, stream);
}

int64_t matmul_weight_copies(const MatmulWeight& p) { return p.rows != nullptr ? weight_copies(p).bytes : 0; }

cudaError_t launch_matmul_weight(const MatmulWeight& p, int device, cudaStream_t stream) {
  if (refused(p.m, p.n, p.k, p.groups, device) || p.m < 1 || p.k % 8 || p.dz_ld % 8) return cudaErrorInvalidValue;
  PairArgs a{};
  a.rows = p.rows;
  a.groups = p.rows ? p.groups : 1;
  a.n_rows = (int)p.m;
  a.features = (int)p.k;
  a.result_rows = (int)p.n;
  a.wide = fours(p.db, p.k, p.type);
  a.idesc = sm100::umma_idesc_16(p.type == Type::kBf16, true, true);
  a.e.out = p.db;
  a.e.most = p.most;
  a.e.out_ld = p.k;
  a.e.n = (int)p.k;
  a.e.type = p.type;
  PairMaps maps{};
  const WeightCopies c = weight_copies(p);
  uint8_t* of_dz = static_cast<uint8_t*>(p.copies) + c.a_bytes;
  auto map = [](CUtensorMap* m, int chunks, const void* base, int64_t rows, int64_t cols, int64_t ld) {
    return chunks == 2 ? map_chunks(m, base, rows, cols, ld, kPairK) : map_2d(m, base, rows, cols, ld, kPairK);
  };
  int n_sm = 0;
  cudaError_t err = multiprocessors(device, &n_sm);
  if (err != cudaSuccess) return err;
  const int steps = weight_steps(p.n, p.m, a.groups, (p.k + kPairM - 1) / kPairM, n_sm);
  a.p_chunks = p.k % kChunk == 0 && p.k > kChunk ? 2 : 1;
  a.q_chunks = p.n % kPairN == 0 && steps == kPairN / kWeightStep ? 2 : 1;  // every tile has 256 result rows
  err = map(&maps.p[0], a.p_chunks, p.a, p.m, p.k, p.a_ld);
  if (err == cudaSuccess) err = map(&maps.q[0], a.q_chunks, p.dz, p.m, p.n, p.dz_ld);
  if (p.rows != nullptr) {
    if (p.copies == nullptr) return cudaErrorInvalidValue;
    a.copies = 1;
    if (err == cudaSuccess) err = map(&maps.p[1], a.p_chunks, p.copies, (int64_t)a.groups * kPairK, p.k, c.a_ld);
    if (err == cudaSuccess) err = map(&maps.q[1], a.q_chunks, of_dz, (int64_t)a.groups * kPairK, p.n, c.dz_ld);
    LastBlocks l{};
    l.from[0] = p.a, l.from[1] = p.dz;
    l.to[0] = p.copies, l.to[1] = of_dz;
    l.from_ld[0] = p.a_ld * 2, l.from_ld[1] = p.dz_ld * 2;
    l.to_ld[0] = c.a_ld * 2, l.to_ld[1] = c.dz_ld * 2;
    l.words[0] = (int)(c.a_ld / 8), l.words[1] = (int)(c.dz_ld / 8);
    l.bytes[0] = p.k * 2, l.bytes[1] = p.n * 2;
    l.rows = p.rows;
    l.groups = a.groups;
    l.m = (int)p.m;
    const int words = l.words[0] + l.words[1];
    auto kernel = last_blocks_kernel;
    if (err == cudaSuccess) err = launch_after(kernel, dim3((words + 255) / 256, a.groups, 4), dim3(256), 0, stream, l);
  }
  return err != cudaSuccess ? err : launch_pairs<kWeight>(maps, a, device, stream);
}

cudaError_t matmul_pre_parts(const MatmulPre& p, int device, int64_t* floats, int* splits) {
  int n_sm = 0;
  cudaError_t err = multiprocessors(device, &n_sm);
  if (err != cudaSuccess) return err;
  // about eight CTAs per SM, no part of less than 32 rows on average
  const int64_t groups = p.rows ? p.groups : 1, columns = (p.n + kPreColumns - 1) / kPreColumns;
  int64_t parts = (8 * (int64_t)n_sm + columns * groups - 1) / (columns * groups);
  const int64_t most = p.m / groups / 32;
  if (parts > most) parts = most;
  if (parts < 1) parts = 1;
  *splits = (int)parts;
  *floats = p.dbias != nullptr && parts > 1 ? groups * parts * p.n : 0;
  return cudaSuccess;
}

cudaError_t launch_matmul_pre(const MatmulPre& p, int device, cudaStream_t stream) {
  if (refused(p.m, p.n, 1, p.groups, device) || (p.activation == kSwiglu && p.n % (2 * kGateBlock))) return cudaErrorInvalidValue;
  int64_t floats = 0;
  PreArgs a = pre_args(p);
  cudaError_t err = matmul_pre_parts(p, device, &floats, &a.splits);
  if (err != cudaSuccess) return err;
  if (floats == 0) a.parts = nullptr;
  else if (a.parts == nullptr) return cudaErrorInvalidValue;
  const bool vec = p.n % 4 == 0 && fours(p.dout, p.dout_ld, p.out_type) && fours(p.pre, p.pre_ld, Type::kF32) && fours(p.dz, p.dz_ld, p.type) &&
                   fours(p.dz_weight, p.dz_ld, p.type);
  const dim3 grid((unsigned)((p.n + kPreColumns - 1) / kPreColumns), (unsigned)a.splits, (unsigned)a.groups);
  const bool gated = p.activation == kSwiglu;
  const bool in_parts = p.row_most != nullptr || p.column_most != nullptr;
  auto pass = [&](auto which) {
    constexpr Pass kPass = decltype(which)::value;
    auto kernel = gated ? vec ? pre_gradient_kernel<true, true, kPass> : pre_gradient_kernel<false, true, kPass>
                        : vec ? pre_gradient_kernel<true, false, kPass> : pre_gradient_kernel<false, false, kPass>;
    return launch_after(kernel, grid, dim3(256), 0, stream, a);
  };
  if (in_parts) {
    const int64_t n_rows = p.row_most != nullptr ? p.m : 0, n_columns = p.column_most != nullptr ? (int64_t)a.groups * p.n : 0;
    auto clear = clear_most_kernel;
    const int64_t longer = n_rows > n_columns ? n_rows : n_columns;
    err = launch_after(clear, dim3((unsigned)((longer + 255) / 256)), dim3(256), 0, stream, p.row_most, n_rows, p.column_most, n_columns);
    if (err == cudaSuccess) err = pass(std::integral_constant<Pass, kMost>{});
    PreArgs sums = a;
    a.parts = nullptr, a.dbias = nullptr;
    if (err == cudaSuccess) err = pass(std::integral_constant<Pass, kParts>{});
    a = sums;
  } else {
    err = pass(std::integral_constant<Pass, kOnePass>{});
  }
  if (err != cudaSuccess || floats == 0) return err;
  const int64_t total = (int64_t)a.groups * a.n;
  auto sum = bias_parts_kernel;
  return launch_after(sum, dim3((unsigned)((total + 255) / 256)), dim3(256), 0, stream, a.parts, a.dbias, a.bias_type, (int64_t)a.n, a.splits,
                      total);
}

}  // namespace ops
}  // namespace lplb

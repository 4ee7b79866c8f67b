// Rows sorted by expert and back.
//
// expert_order   a stable counting sort of the pairs (token, choice) by expert
// take_rows      rows[place[t, k]] = x[t]
// combine_rows   out[t] = sum over k of w[t, k] rows[place[t, k]], in 32 bits, in the order of k
//                drows[place[t, k]] = w[t, k] dout[t],   dw[t, k] = <dout[t], rows[place[t, k]]>
//
// take_rows and combine_rows without weights are each other's gradient.  All three go by token, not by sorted row: the token's side is
// read or written once, and its rows, which lie far apart but are each of one piece, all at once.  Bound by DRAM; nothing is summed
// by atomics, the same inputs give the same bits.  What decided their speed: few enough registers for three or four CTAs per SM, and no branch
// between a thread's loads.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <initializer_list>
#include <type_traits>

#include "common.cuh"
#include "experts_api.h"
#include "tcgen05.cuh"

namespace lplb {
namespace ops {
namespace {

constexpr uint32_t kAll = 0xffffffffu;

// ---- the order ------------------------------------------------------------------------------------
// One cluster of up to 16 CTAs sorts all pairs.  Every warp counts a stretch of consecutive pairs per expert, in shared memory of
// its own; the counts of the warps and CTAs before it, and of the experts before, are where its pairs begin; then it goes through
// its stretch again, 32 pairs at a time, and lanes with the same expert take consecutive places in the order of lanes.
constexpr int kOrderThreads = 1024, kOrderWarps = kOrderThreads / 32, kOrderMaxCluster = 16;
constexpr int kBatch = 8;  // loads of 32 pairs under way

size_t order_smem(int warps, int experts) { return (size_t)(warps + 2) * experts * sizeof(uint32_t); }

__device__ __forceinline__ uint32_t ld_cluster(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

template <typename I>
__global__ void __launch_bounds__(kOrderThreads) order_kernel(const Order o, int warps, int64_t stretch) {
  using namespace sm100;
  extern __shared__ uint32_t order_shared[];
  uint32_t* hist = order_shared;           // [warps][experts]
  uint32_t* total = hist + warps * o.experts;  // [experts] this CTA's pairs
  uint32_t* base = total + o.experts;      // [experts] place of this CTA's first pair
  __shared__ uint32_t part[kOrderWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;
  const int rank = (int)cluster_cta_rank(), ctas = (int)cluster_size();
  const I* idx = static_cast<const I*>(o.idx);
  for (int i = tid; i < warps * o.experts; i += kOrderThreads) hist[i] = 0;
  __syncthreads();
  wait_predecessors();
  allow_successor();
  // this warp's stretch, a multiple of 32 pairs
  int64_t from = o.pairs, to = o.pairs;
  if (warp < warps) {
    from = min(o.pairs, ((int64_t)rank * warps + warp) * stretch);
    to = min(o.pairs, from + stretch);
  }
  uint32_t* mine = hist + warp * o.experts;
  int e[kBatch];
  auto each = [&](auto&& use, bool kept) {  // 32 pairs at a time: the pair and its expert, -1 where there is none
    for (int64_t at = from; at < to; at += 32 * kBatch) {
      if (!kept) {  // (a stretch of one batch stays in registers for the second time)
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          const int64_t p = at + 32 * i + lane;
          const long long v = p < to ? (long long)idx[p] : -1;
          e[i] = v >= 0 && v < o.experts ? (int)v : -1;
        }
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
        if (at + 32 * i < to) use(at + 32 * i + lane, e[i]);
    }
  };
  each([&](int64_t, int e) {
    if (e >= 0) atomicAdd(&mine[e], 1u);
  }, false);
  __syncthreads();
  for (int e = tid; e < o.experts; e += kOrderThreads) {
    uint32_t run = 0;
    for (int w = 0; w < warps; ++w) {
      const uint32_t n = hist[w * o.experts + e];
      hist[w * o.experts + e] = run;
      run += n;
    }
    total[e] = run;
  }
  if (ctas > 1) cluster_sync();
  else __syncthreads();
  // an expert per thread: pairs of the CTAs before this one, of all, and of the experts before
  uint32_t before = 0, all = 0;
  if (tid < o.experts) {
    const uint32_t at = smem_u32(&total[tid]);
    uint32_t n[kOrderMaxCluster];
#pragma unroll
    for (int r = 0; r < kOrderMaxCluster; ++r) n[r] = r < ctas ? ld_cluster(map_to_rank(at, r)) : 0;
#pragma unroll
    for (int r = 0; r < kOrderMaxCluster; ++r) {
      if (r < rank) before += n[r];
      all += n[r];
    }
    if (rank == 0) o.counts[tid] = (int)all;
  }
  uint32_t scan = all;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t v = __shfl_up_sync(kAll, scan, d);
    if (lane >= d) scan += v;
  }
  if (lane == 31) part[warp] = scan;
  __syncthreads();
  uint32_t sum = part[lane], upto = sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t v = __shfl_up_sync(kAll, upto, d);
    if (lane >= d) upto += v;
  }
  const uint32_t used = __shfl_sync(kAll, upto, 31);
  const uint32_t warps_before = warp ? __shfl_sync(kAll, upto, warp - 1) : 0;
  if (tid < o.experts) base[tid] = warps_before + scan - all + before;
  __syncthreads();
  each([&](int64_t p, int e) {
    const uint32_t same = __match_any_sync(kAll, e);
    uint32_t at = 0;
    if (e >= 0) at = base[e] + mine[e] + __popc(same & ((1u << lane) - 1));
    __syncwarp();
    if (e >= 0 && lane == __ffs(same) - 1) mine[e] += __popc(same);
    __syncwarp();
    if (p < to) {
      o.place[p] = e >= 0 ? (int)at : -1;
      if (e >= 0) o.source[at] = (int)p;
    }
  }, to - from <= 32 * kBatch);
  for (int64_t r = used + (int64_t)rank * kOrderThreads + tid; r < o.pairs; r += (int64_t)ctas * kOrderThreads) o.source[r] = -1;
  if (ctas > 1) cluster_sync();  // nobody leaves while another reads its totals
}

// ---- geometry of the kernels that go by token ---------------------------------------------------
// A token's row is dealt out, in vectors, to the threads of `x`; a CTA has `y` tokens, and `splits` CTAs share a token's row
// where there are so few tokens that the SMs would stay empty.
struct Shape {
  dim3 grid, block;
};
Shape shape_of(int64_t tokens, int64_t vectors, int per_thread, int n_sms, bool whole_rows) {
  int64_t threads = (vectors + per_thread - 1) / per_thread;
  threads = threads < 32 ? 32 : threads > 256 ? 256 : (threads + 31) / 32 * 32;
  const int64_t y = whole_rows && threads > 32 ? 1 : 256 / threads;
  const int64_t x = (tokens + y - 1) / y;
  int64_t splits = 1;
  if (!whole_rows) {
    const int64_t most = (vectors + threads - 1) / threads;
    splits = (4 * (int64_t)n_sms + x - 1) / x;
    if (splits > most) splits = most;
    if (splits < 1) splits = 1;
  }
  return {dim3((unsigned)x, (unsigned)splits), dim3((unsigned)threads, (unsigned)y)};
}

template <int N>
struct Bytes;
template <> struct Bytes<16> { using type = uint4; };
template <> struct Bytes<8> { using type = uint2; };
template <> struct Bytes<4> { using type = uint32_t; };
template <> struct Bytes<2> { using type = uint16_t; };
template <> struct Bytes<1> { using type = uint8_t; };

// ---- rows to their experts ------------------------------------------------------------------------
// us, 8192 tokens x 8 rows of 7168 in bf16: 171 (6.2 TB/s).  By bulk copies through shared memory, a row loaded once and stored eight times, 186.
constexpr int kTakeVectors = 4;  // of a row, per thread and round
template <int N>
__global__ void __launch_bounds__(256, 4) take_rows_kernel(const TakeRows a) {
  using V = typename Bytes<N>::type;
  wait_predecessors();
  allow_successor();
  const int64_t token = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (token >= a.tokens) return;
  const int64_t vectors = a.row_bytes / N, n_rows = a.tokens * a.topk;
  const V* x = reinterpret_cast<const V*>(static_cast<const uint8_t*>(a.x) + token * a.ld_bytes);
  V* rows = static_cast<V*>(a.rows);
  const int* place = a.place + token * a.topk;
  const int* source = a.source + token * a.topk;
  const int64_t step = (int64_t)gridDim.y * blockDim.x;
  for (int64_t v0 = (int64_t)blockIdx.y * blockDim.x + threadIdx.x; v0 < vectors; v0 += step * kTakeVectors) {
    V v[kTakeVectors];
#pragma unroll
    for (int i = 0; i < kTakeVectors; ++i) v[i] = v0 + i * step < vectors ? x[v0 + i * step] : V{};
    auto put = [&](int64_t row, const V (&what)[kTakeVectors]) {
      V* to = rows + row * vectors + v0;
#pragma unroll
      for (int i = 0; i < kTakeVectors; ++i)
        if (v0 + i * step < vectors) to[i * step] = what[i];
    };
    const V zero[kTakeVectors]{};
#pragma unroll 4
    for (int k = 0; k < a.topk; ++k) {
      const int64_t to = place[k];
      if (to >= 0 && to < n_rows) put(to, v);
    }
#pragma unroll 4
    for (int k = 0; k < a.topk; ++k)
      if (source[k] < 0) put(token * a.topk + k, zero);  // a row that nobody has
  }
}

// ---- and back ---------------------------------------------------------------------------------------
// N neighbouring values of a row, in registers as they are in memory
template <typename T, int N>
struct alignas(sizeof(T) * N) Few {
  T v[N];
};
// in one piece
template <typename T, int N>
__device__ __forceinline__ Few<T, N> load_few(const T* p) {
  using Raw = typename Bytes<sizeof(T) * N>::type;
  const Raw raw = *reinterpret_cast<const Raw*>(p);
  Few<T, N> f;
  *reinterpret_cast<Raw*>(&f) = raw;
  return f;
}
template <typename T, int N>
__device__ __forceinline__ void store_few(T* p, const Few<T, N>& f) {
  using Raw = typename Bytes<sizeof(T) * N>::type;
  *reinterpret_cast<Raw*>(p) = *reinterpret_cast<const Raw*>(&f);
}
__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
__device__ __forceinline__ void narrow(float& p, float v) { p = v; }
__device__ __forceinline__ void narrow(__nv_bfloat16& p, float v) { p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void narrow(__half& p, float v) { p = __float2half_rn(v); }

// Vectors of a row per thread and round: 16 bytes, of rows off 4 bytes 8 (8192 x 8 rows of 2051 in bf16 back 102 us, with 16 bytes 124).
template <typename T, int N>
constexpr int kVectorsOf = N * sizeof(T) == 2 ? 4 : 16 / (N * sizeof(T));

// ROWS of a token's rows at vectors v0, v0 + step, ... of their columns.  Nothing is asked between the loads (each would wait for the one
// before): what is not there is read from the first row, or the row's first vector, and left out by the caller.
template <int ROWS, int VECTORS, typename T, int N>
__device__ __forceinline__ void load_rows(const T* rows, int64_t ld, const int64_t (&at)[ROWS], int v0, int step, int vectors, Few<T, N> (&y)[ROWS][VECTORS]) {
#pragma unroll
  for (int j = 0; j < ROWS; ++j) {
    const T* from = rows + (at[j] < 0 ? 0 : at[j]) * ld;
#pragma unroll
    for (int v = 0; v < VECTORS; ++v) y[j][v] = load_few<T, N>(from + (int64_t)(v0 + v * step < vectors ? v0 + v * step : 0) * N);
  }
}

// us, 8192 tokens x 8, 2, 1 rows of 7168 in bf16: 172, 78, 51 (6.1 TB/s at 8); with four rows at a time whatever is left 178, 82, 57.  Bulk copies into
// shared memory, 190 KB per SM under way, took 195, 104 and 84.
template <typename T, int N>
__global__ void __launch_bounds__(256, 4) combine_rows_kernel(const CombineRows a) {
  constexpr int kVectors = kVectorsOf<T, N>;
  wait_predecessors();
  allow_successor();
  const int64_t token = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (token >= a.tokens) return;
  const int64_t n_rows = a.tokens * a.topk;
  const int vectors = a.cols / N, step = gridDim.y * blockDim.x;
  const T* rows = static_cast<const T*>(a.rows);
  const int* place = a.place + token * a.topk;
  T* out = static_cast<T*>(a.out) + token * a.cols;
  for (int v0 = blockIdx.y * blockDim.x + threadIdx.x; v0 < vectors; v0 += step * kVectors) {
    float sum[kVectors][N];
#pragma unroll
    for (int v = 0; v < kVectors; ++v)
#pragma unroll
      for (int n = 0; n < N; ++n) sum[v][n] = 0.f;
    auto add = [&](int k0, auto count) {
      constexpr int kRows = decltype(count)::value;
      Few<T, N> y[kRows][kVectors];
      float w[kRows];
      int64_t at[kRows];
#pragma unroll
      for (int j = 0; j < kRows; ++j) {
        at[j] = place[k0 + j];
        w[j] = a.weights != nullptr ? a.weights[token * a.topk + k0 + j] : 1.f;
      }
#pragma unroll
      for (int j = 0; j < kRows; ++j)
        if (at[j] >= n_rows) at[j] = -1;
      load_rows<kRows, kVectors>(rows, a.ld, at, v0, step, vectors, y);
#pragma unroll
      for (int j = 0; j < kRows; ++j) {
        if (at[j] < 0) continue;
#pragma unroll
        for (int v = 0; v < kVectors; ++v)
#pragma unroll
          for (int n = 0; n < N; ++n) sum[v][n] = fmaf(w[j], widen(y[j][v].v[n]), sum[v][n]);
      }
    };
    int k = 0;
    for (; k + 4 <= a.topk; k += 4) add(k, std::integral_constant<int, 4>{});
    if (a.topk & 2) add(k, std::integral_constant<int, 2>{}), k += 2;
    if (a.topk & 1) add(k, std::integral_constant<int, 1>{});
#pragma unroll
    for (int v = 0; v < kVectors; ++v) {
      Few<T, N> r;
#pragma unroll
      for (int n = 0; n < N; ++n) narrow(r.v[n], sum[v][n]);
      if (v0 + v * step < vectors) store_few(out + (int64_t)(v0 + v * step) * N, r);
    }
  }
}

// us, as above: 360, 104, 80 (5.5 TB/s at 8); with four rows at a time 353, 137, 116; by bulk copies 346, 180 and 153.
template <typename T, int N>
__global__ void __launch_bounds__(256, 4) combine_rows_backward_kernel(const CombineRows a) {
  constexpr int kVectors = kVectorsOf<T, N>;
  __shared__ float part[2][8];
  wait_predecessors();
  allow_successor();
  const int64_t token = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  if (token >= a.tokens) return;  // a CTA of several warps per token has one token
  const int64_t n_rows = a.tokens * a.topk;
  const int vectors = a.cols / N, step = blockDim.x;
  const T* rows = static_cast<const T*>(a.rows);
  T* drows = static_cast<T*>(a.drows);
  const T* dout = static_cast<const T*>(a.dout) + token * a.dout_ld;
  auto choices = [&](int k0, auto count) {
    constexpr int kRows = decltype(count)::value;
    int64_t at[kRows];
    float w[kRows], dot[kRows];
    bool spare[kRows];
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
      at[j] = a.place[token * a.topk + k0 + j];
      w[j] = a.weights[token * a.topk + k0 + j];
      spare[j] = drows != nullptr && a.source[token * a.topk + k0 + j] < 0;
      dot[j] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < kRows; ++j)
      if (at[j] >= n_rows) at[j] = -1;
    for (int v0 = threadIdx.x; v0 < vectors; v0 += step * kVectors) {
      Few<T, N> d[1][kVectors], y[kRows][kVectors];
      const int64_t first[1] = {0};
      load_rows<1, kVectors>(dout, 0, first, v0, step, vectors, d);
      if (a.dweights != nullptr) load_rows<kRows, kVectors>(rows, a.ld, at, v0, step, vectors, y);
#pragma unroll
      for (int v = 0; v < kVectors; ++v) {
        if (v0 + v * step >= vectors) continue;
        const int64_t column = (int64_t)(v0 + v * step) * N;
#pragma unroll
        for (int j = 0; j < kRows; ++j) {
          if (at[j] >= 0) {
            if (drows != nullptr) {
              Few<T, N> r;
#pragma unroll
              for (int n = 0; n < N; ++n) narrow(r.v[n], w[j] * widen(d[0][v].v[n]));
              store_few(drows + at[j] * a.cols + column, r);
            }
            if (a.dweights != nullptr) {
#pragma unroll
              for (int n = 0; n < N; ++n) dot[j] = fmaf(widen(d[0][v].v[n]), widen(y[j][v].v[n]), dot[j]);
            }
          }
          if (spare[j]) {  // a row that nobody has
            Few<T, N> zero;
#pragma unroll
            for (int n = 0; n < N; ++n) narrow(zero.v[n], 0.f);
            store_few(drows + (token * a.topk + k0 + j) * a.cols + column, zero);
          }
        }
      }
    }
    if (a.dweights == nullptr) return;
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
#pragma unroll
      for (int s = 16; s > 0; s >>= 1) dot[j] += __shfl_xor_sync(kAll, dot[j], s);
    }
    if (warps == 1) {
#pragma unroll
      for (int j = 0; j < kRows; ++j)
        if (lane == j) a.dweights[token * a.topk + k0 + j] = dot[j];
      return;
    }
#pragma unroll
    for (int j = 0; j < kRows; ++j)
      if (lane == j) part[j][warp] = dot[j];
    __syncthreads();
    if (warp == 0 && lane < kRows) {
      float sum = 0.f;
      for (int i = 0; i < warps; ++i) sum += part[lane][i];
      a.dweights[token * a.topk + k0 + lane] = sum;
    }
    __syncthreads();
  };
  int k = 0;
  for (; k + 2 <= a.topk; k += 2) choices(k, std::integral_constant<int, 2>{});
  if (a.topk & 1) choices(k, std::integral_constant<int, 1>{});
}

// The widest vector, in bytes of 16 or less, that divides all of these.
int widest(std::initializer_list<uint64_t> of) {
  uint64_t all = 16;
  for (uint64_t v : of) all |= v;
  return (int)(all & (~all + 1));
}
uint64_t address(const void* p) { return reinterpret_cast<uintptr_t>(p); }

template <int N>
cudaError_t launch_take(const TakeRows& t, int n_sms, cudaStream_t stream) {
  const Shape s = shape_of(t.tokens, t.row_bytes / N, kTakeVectors, n_sms, false);
  auto kernel = take_rows_kernel<N>;
  return launch_after(kernel, s.grid, s.block, 0, stream, t);
}

bool refused(const CombineRows& c) { return c.tokens < 0 || c.tokens > INT32_MAX || c.cols < 1 || c.topk < 1; }

template <typename T, int N>
cudaError_t launch_combine(const CombineRows& c, int n_sms, bool backward, cudaStream_t stream) {
  const int vectors = c.cols / N;
  if (backward) {
    const Shape s = shape_of(c.tokens, vectors, kVectorsOf<T, N>, n_sms, true);
    auto kernel = combine_rows_backward_kernel<T, N>;
    return launch_after(kernel, s.grid, s.block, 0, stream, c);
  }
  const Shape s = shape_of(c.tokens, vectors, kVectorsOf<T, N>, n_sms, false);
  auto kernel = combine_rows_kernel<T, N>;
  return launch_after(kernel, s.grid, s.block, 0, stream, c);
}
template <typename T>
cudaError_t launch_combine(const CombineRows& c, int n_sms, bool backward, cudaStream_t stream) {
  const uint64_t size = sizeof(T);
  int wide = backward ? widest({address(c.rows), c.ld * size, c.cols * size, address(c.dout), c.dout_ld * size, address(c.drows)})
                      : widest({address(c.rows), c.ld * size, c.cols * size, address(c.out)});
  if (wide == 16) return launch_combine<T, 16 / sizeof(T)>(c, n_sms, backward, stream);
  if (wide >= 4) return launch_combine<T, 4 / sizeof(T)>(c, n_sms, backward, stream);
  if constexpr (sizeof(T) == 2) return launch_combine<T, 1>(c, n_sms, backward, stream);
  return cudaErrorMisalignedAddress;
}
cudaError_t launch_combine(const CombineRows& c, int n_sms, bool backward, cudaStream_t stream) {
  if (refused(c)) return cudaErrorInvalidValue;
  if (c.tokens == 0) return cudaSuccess;
  switch (c.type) {
    case Type::kF32: return launch_combine<float>(c, n_sms, backward, stream);
    case Type::kBf16: return launch_combine<__nv_bfloat16>(c, n_sms, backward, stream);
    default: return launch_combine<__half>(c, n_sms, backward, stream);
  }
}

// Whether a cluster of kOrderMaxCluster CTAs, which is more than every device promises, can run here.
cudaError_t largest_cluster_fits(int device, int* fits) {
  static std::atomic<int> known[kMaxDevices];  // 1: no, 2: yes
  if (known[device].load(std::memory_order_relaxed) == 0) {
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = kOrderMaxCluster;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(kOrderMaxCluster);
    config.blockDim = dim3(kOrderThreads);
    config.dynamicSmemBytes = order_smem(kOrderWarps, kOrderMaxExperts);
    config.attrs = &attr;
    config.numAttrs = 1;
    int clusters = 0;
    const cudaError_t err = cudaOccupancyMaxActiveClusters(&clusters, order_kernel<int64_t>, &config);
    if (err != cudaSuccess) return err;
    known[device].store(clusters > 0 ? 2 : 1, std::memory_order_relaxed);
  }
  *fits = known[device].load(std::memory_order_relaxed) == 2;
  return cudaSuccess;
}

}  // namespace

cudaError_t launch_order(const Order& o, int device, cudaStream_t stream) {
  if (o.pairs < 0 || o.pairs > INT32_MAX || o.experts < 1 || o.experts > kOrderMaxExperts) return cudaErrorInvalidValue;
  auto kernel = o.is64 ? order_kernel<int64_t> : order_kernel<int32_t>;
  static std::atomic<bool> prepared[kMaxDevices];
  if (device < 0 || device >= kMaxDevices) return cudaErrorInvalidDevice;
  if (!prepared[device].load(std::memory_order_relaxed)) {
    const int most = (int)order_smem(kOrderWarps, kOrderMaxExperts);
    cudaError_t err = cudaFuncSetAttribute(order_kernel<int64_t>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    if (err == cudaSuccess) err = cudaFuncSetAttribute(order_kernel<int32_t>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    if (err == cudaSuccess) err = cudaFuncSetAttribute(order_kernel<int64_t>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (err == cudaSuccess) err = cudaFuncSetAttribute(order_kernel<int32_t>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (err != cudaSuccess) return err;
    prepared[device].store(true, std::memory_order_relaxed);
  }
  // a CTA up to 64 chunks of 32 pairs, then as many as give each that many, where the device has room for such a cluster
  const int64_t chunks = (o.pairs + 31) / 32;
  int ctas = 1;
  while (ctas < kOrderMaxCluster && ctas * 64 < chunks) ctas *= 2;
  if (ctas > 8) {
    int fit = 0;
    const cudaError_t err = largest_cluster_fits(device, &fit);
    if (err != cudaSuccess) return err;
    if (!fit) ctas = 8;
  }
  int warps = (int)((chunks + ctas - 1) / ctas);
  if (warps > kOrderWarps) warps = kOrderWarps;
  if (warps < 1) warps = 1;
  const int64_t stretch = (chunks + (int64_t)ctas * warps - 1) / ((int64_t)ctas * warps) * 32;
  cudaLaunchAttribute attrs[2]{};
  attrs[0].id = cudaLaunchAttributeClusterDimension;
  attrs[0].val.clusterDim.x = ctas;
  attrs[0].val.clusterDim.y = attrs[0].val.clusterDim.z = 1;
  attrs[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(ctas);
  config.blockDim = dim3(kOrderThreads);
  config.dynamicSmemBytes = order_smem(warps, o.experts);
  config.stream = stream;
  config.attrs = attrs;
  config.numAttrs = 2;
  return cudaLaunchKernelEx(&config, kernel, o, warps, stretch);
}

cudaError_t launch_take_rows(const TakeRows& t, int n_sms, cudaStream_t stream) {
  if (t.tokens < 0 || t.tokens > INT32_MAX || t.row_bytes < 1 || t.topk < 1) return cudaErrorInvalidValue;
  if (t.tokens == 0) return cudaSuccess;
  switch (widest({address(t.x), (uint64_t)t.ld_bytes, (uint64_t)t.row_bytes, address(t.rows)})) {
    case 16: return launch_take<16>(t, n_sms, stream);
    case 8: return launch_take<8>(t, n_sms, stream);
    case 4: return launch_take<4>(t, n_sms, stream);
    case 2: return launch_take<2>(t, n_sms, stream);
    default: return launch_take<1>(t, n_sms, stream);
  }
}

cudaError_t launch_combine_rows(const CombineRows& c, int n_sms, cudaStream_t stream) { return launch_combine(c, n_sms, false, stream); }
cudaError_t launch_combine_rows_backward(const CombineRows& c, int n_sms, cudaStream_t stream) { return launch_combine(c, n_sms, true, stream); }

}  // namespace ops
}  // namespace lplb

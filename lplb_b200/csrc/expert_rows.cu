// Rows sorted by expert and back.
//
// expert_order   a stable counting sort of the pairs (token, choice) by expert
// take_rows      rows[place[t, k]] = x[t]
// combine_rows   out[t] = sum over k of w[t, k] rows[place[t, k]], in 32 bits, in the order of k
//                drows[place[t, k]] = w[t, k] dout[t],   dw[t, k] = <dout[t], rows[place[t, k]]>
//
// take_rows and combine_rows without weights are each other's gradient.  All three go by token, not by sorted row: the token's side is
// read or written once, and its rows, which lie far apart but are each of one piece, all at once.  Bound by DRAM; nothing is summed
// by atomics, the same inputs give the same bits.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <initializer_list>

#include "common.cuh"
#include "experts_api.h"
#include "tcgen05.cuh"

namespace lplb {
namespace ops {
namespace {

constexpr uint32_t kAll = 0xffffffffu;

// ---- the order ------------------------------------------------------------------------------------
// One cluster of up to 8 CTAs sorts all pairs.  Every warp counts a stretch of consecutive pairs per expert, in shared memory of
// its own; the counts of the warps and CTAs before it, and of the experts before, are where its pairs begin; then it goes through
// its stretch again, 32 pairs at a time, and lanes with the same expert take consecutive places in the order of lanes.
constexpr int kOrderThreads = 1024, kOrderWarps = kOrderThreads / 32, kOrderMaxCluster = 8;
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
  allow_successor();
  for (int i = tid; i < warps * o.experts; i += kOrderThreads) hist[i] = 0;
  __syncthreads();
  wait_predecessors();
  // this warp's stretch, a multiple of 32 pairs
  int64_t from = o.pairs, to = o.pairs;
  if (warp < warps) {
    from = min(o.pairs, ((int64_t)rank * warps + warp) * stretch);
    to = min(o.pairs, from + stretch);
  }
  uint32_t* mine = hist + warp * o.experts;
  auto each = [&](auto&& use) {  // 32 pairs at a time: the pair and its expert, -1 where there is none
    for (int64_t at = from; at < to; at += 32 * kBatch) {
      int e[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int64_t p = at + 32 * i + lane;
        const long long v = p < to ? (long long)idx[p] : -1;
        e[i] = v >= 0 && v < o.experts ? (int)v : -1;
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
        if (at + 32 * i < to) use(at + 32 * i + lane, e[i]);
    }
  };
  each([&](int64_t, int e) {
    if (e >= 0) atomicAdd(&mine[e], 1u);
  });
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
  });
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

constexpr int kRowsAtOnce = 8;  // of a token

// ---- rows to their experts ------------------------------------------------------------------------
constexpr int kTakeVectors = 4;  // of a row, per thread and round
template <int N>
__global__ void __launch_bounds__(256) take_rows_kernel(const TakeRows a) {
  using V = typename Bytes<N>::type;
  allow_successor();
  wait_predecessors();
  const int64_t token = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (token >= a.tokens) return;
  const int64_t vectors = a.row_bytes / N, n_rows = a.tokens * a.topk;
  const V* x = reinterpret_cast<const V*>(static_cast<const uint8_t*>(a.x) + token * a.ld_bytes);
  V* rows = static_cast<V*>(a.rows);
  const int64_t step = (int64_t)gridDim.y * blockDim.x;
  const V zero{};
  for (int64_t v0 = (int64_t)blockIdx.y * blockDim.x + threadIdx.x; v0 < vectors; v0 += step * kTakeVectors) {
    V v[kTakeVectors];
#pragma unroll
    for (int i = 0; i < kTakeVectors; ++i) v[i] = v0 + i * step < vectors ? x[v0 + i * step] : zero;
    for (int k0 = 0; k0 < a.topk; k0 += kRowsAtOnce) {
      int place[kRowsAtOnce], source[kRowsAtOnce];
#pragma unroll
      for (int j = 0; j < kRowsAtOnce; ++j) {
        const bool in = k0 + j < a.topk;
        place[j] = in ? a.place[token * a.topk + k0 + j] : -1;
        source[j] = in ? a.source[token * a.topk + k0 + j] : 0;
      }
#pragma unroll
      for (int j = 0; j < kRowsAtOnce; ++j) {
        if (place[j] >= 0 && place[j] < n_rows) {
          V* to = rows + place[j] * vectors;
#pragma unroll
          for (int i = 0; i < kTakeVectors; ++i)
            if (v0 + i * step < vectors) to[v0 + i * step] = v[i];
        }
        if (source[j] < 0) {  // a row that nobody has
          V* to = rows + (token * a.topk + k0 + j) * vectors;
#pragma unroll
          for (int i = 0; i < kTakeVectors; ++i)
            if (v0 + i * step < vectors) to[v0 + i * step] = zero;
        }
      }
    }
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

template <typename T, int N>
__global__ void __launch_bounds__(256) combine_rows_kernel(const CombineRows a) {
  using V = Few<T, N>;
  allow_successor();
  wait_predecessors();
  const int64_t token = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (token >= a.tokens) return;
  const int64_t n_rows = a.tokens * a.topk;
  const int vectors = a.cols / N, step = gridDim.y * blockDim.x;
  const T* rows = static_cast<const T*>(a.rows);
  T* out = static_cast<T*>(a.out) + token * a.cols;
  for (int v0 = blockIdx.y * blockDim.x + threadIdx.x; v0 < vectors; v0 += step) {
    float sum[N];
#pragma unroll
    for (int n = 0; n < N; ++n) sum[n] = 0.f;
    for (int k0 = 0; k0 < a.topk; k0 += kRowsAtOnce) {
      int place[kRowsAtOnce];
      float w[kRowsAtOnce];
      V y[kRowsAtOnce];
#pragma unroll
      for (int j = 0; j < kRowsAtOnce; ++j) {
        const bool in = k0 + j < a.topk;
        place[j] = in ? a.place[token * a.topk + k0 + j] : -1;
        w[j] = in && a.weights != nullptr ? a.weights[token * a.topk + k0 + j] : 1.f;
        if (place[j] >= n_rows) place[j] = -1;
      }
#pragma unroll
      for (int j = 0; j < kRowsAtOnce; ++j)
        if (place[j] >= 0) y[j] = load_few<T, N>(rows + place[j] * a.ld + (int64_t)v0 * N);
#pragma unroll
      for (int j = 0; j < kRowsAtOnce; ++j) {
        if (place[j] < 0) continue;
#pragma unroll
        for (int n = 0; n < N; ++n) sum[n] = fmaf(w[j], widen(y[j].v[n]), sum[n]);
      }
    }
    V r;
#pragma unroll
    for (int n = 0; n < N; ++n) narrow(r.v[n], sum[n]);
    store_few(out + (int64_t)v0 * N, r);
  }
}

template <typename T, int N>
__global__ void __launch_bounds__(256) combine_rows_backward_kernel(const CombineRows a) {
  using V = Few<T, N>;
  __shared__ float part[kRowsAtOnce][8];
  allow_successor();
  wait_predecessors();
  const int64_t token = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  if (token >= a.tokens) return;  // a CTA of several warps per token has one token
  const int64_t n_rows = a.tokens * a.topk;
  const int vectors = a.cols / N;
  const T* rows = static_cast<const T*>(a.rows);
  T* drows = static_cast<T*>(a.drows);
  const T* dout = static_cast<const T*>(a.dout) + token * a.dout_ld;
  for (int k0 = 0; k0 < a.topk; k0 += kRowsAtOnce) {
    int place[kRowsAtOnce];
    float w[kRowsAtOnce], dot[kRowsAtOnce];
    bool spare[kRowsAtOnce];
#pragma unroll
    for (int j = 0; j < kRowsAtOnce; ++j) {
      const bool in = k0 + j < a.topk;
      place[j] = in ? a.place[token * a.topk + k0 + j] : -1;
      w[j] = in ? a.weights[token * a.topk + k0 + j] : 0.f;
      spare[j] = in && drows != nullptr && a.source[token * a.topk + k0 + j] < 0;
      dot[j] = 0.f;
      if (place[j] >= n_rows) place[j] = -1;
    }
    for (int v0 = threadIdx.x; v0 < vectors; v0 += blockDim.x) {
      const V d = load_few<T, N>(dout + (int64_t)v0 * N);
      V y[kRowsAtOnce];
      if (a.dweights != nullptr) {
#pragma unroll
        for (int j = 0; j < kRowsAtOnce; ++j)
          if (place[j] >= 0) y[j] = load_few<T, N>(rows + place[j] * a.ld + (int64_t)v0 * N);
      }
#pragma unroll
      for (int j = 0; j < kRowsAtOnce; ++j) {
        if (place[j] >= 0) {
          if (drows != nullptr) {
            V r;
#pragma unroll
            for (int n = 0; n < N; ++n) narrow(r.v[n], w[j] * widen(d.v[n]));
            store_few(drows + (int64_t)place[j] * a.cols + (int64_t)v0 * N, r);
          }
          if (a.dweights != nullptr) {
#pragma unroll
            for (int n = 0; n < N; ++n) dot[j] = fmaf(widen(d.v[n]), widen(y[j].v[n]), dot[j]);
          }
        }
        if (spare[j]) {
          V zero;
#pragma unroll
          for (int n = 0; n < N; ++n) narrow(zero.v[n], 0.f);
          store_few(drows + (token * a.topk + k0 + j) * a.cols + (int64_t)v0 * N, zero);
        }
      }
    }
    if (a.dweights == nullptr) continue;
#pragma unroll
    for (int j = 0; j < kRowsAtOnce; ++j) {
#pragma unroll
      for (int s = 16; s > 0; s >>= 1) dot[j] += __shfl_xor_sync(kAll, dot[j], s);
    }
    if (warps == 1) {
#pragma unroll
      for (int j = 0; j < kRowsAtOnce; ++j)
        if (lane == j && k0 + j < a.topk) a.dweights[token * a.topk + k0 + j] = dot[j];
      continue;
    }
#pragma unroll
    for (int j = 0; j < kRowsAtOnce; ++j)
      if (lane == j) part[j][warp] = dot[j];
    __syncthreads();
    if (warp == 0 && lane < kRowsAtOnce && k0 + lane < a.topk) {
      float sum = 0.f;
      for (int i = 0; i < warps; ++i) sum += part[lane][i];
      a.dweights[token * a.topk + k0 + lane] = sum;
    }
    __syncthreads();
  }
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
  return launch_after(take_rows_kernel<N>, s.grid, s.block, 0, stream, t);
}

bool refused(const CombineRows& c) { return c.tokens < 0 || c.tokens > INT32_MAX || c.cols < 1 || c.topk < 1; }

template <typename T, int N>
cudaError_t launch_combine(const CombineRows& c, int n_sms, bool backward, cudaStream_t stream) {
  const int vectors = c.cols / N;
  if (backward) {
    const Shape s = shape_of(c.tokens, vectors, 2, n_sms, true);
    return launch_after(combine_rows_backward_kernel<T, N>, s.grid, s.block, 0, stream, c);
  }
  const Shape s = shape_of(c.tokens, vectors, 1, n_sms, false);
  return launch_after(combine_rows_kernel<T, N>, s.grid, s.block, 0, stream, c);
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
    if (err != cudaSuccess) return err;
    prepared[device].store(true, std::memory_order_relaxed);
  }
  // a CTA up to 64 chunks of 32 pairs, then as many as give each that many
  const int64_t chunks = (o.pairs + 31) / 32;
  int ctas = 1;
  while (ctas < kOrderMaxCluster && ctas * 64 < chunks) ctas *= 2;
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
cudaError_t launch_combine_rows_backward(const CombineRows& c, cudaStream_t stream) { return launch_combine(c, 1, true, stream); }

}  // namespace ops
}  // namespace lplb

// Rows to 8 bits, with the residual's addition and the root-mean-square norm in front.
//
//   h = round(x + r)            to x's type: the sum is an output, and what the next layer sees is normed
//   n = h * w / sqrt(mean(h^2) + eps)
//   s = 2^ceil(log2(max|n| / 448))   per block of 128,   q = e4m3(n / s)
//
// One pass: a row's values stay in registers between the sum of squares and the conversion, so x, r
// and w are read once and h, q and s written once.  Everything between is in 32 bits.  Bound by issue slots and DRAM
// at once: 8192 rows of 7168 in bf16 with a residual 82-86 us, 4.9 TB/s (2.6 instructions a cycle), in float32 155-161; converted
// only 36; 4 rows 2.4 us.
#include "ops_api.h"

#include "common.cuh"
#include "fp8.cuh"

namespace lplb {
namespace ops {
namespace {

using namespace fp8;

// A row belongs to blockDim.x threads (whole warps), every thread to V vectors of eight values that are
// blockDim.x vectors apart; 16 neighbouring lanes hold a block of 128.  Rows of one warp share a CTA.
//
// The norm's factor is the same for a row, so the scale is found from h * w, times that factor, and the conversion multiplies
// by the factor over the scale: scaling by powers of two rounds nothing.

// h * w and the sum's place in the chain: values, e4m3 and scale of one vector
template <typename T, bool NORM, bool VEC>
__device__ __forceinline__ void finish(const RowFp8& a, float2 (&v)[4], const float2 (&w)[4], float inv, int64_t row, int c, int n, int blocks) {
  if (NORM) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = mul2(v[i], w[i]);
    if (a.normed != nullptr) {
      float2 f[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = mul2(v[i], make_float2(inv, inv));
      store_raw<VEC>(static_cast<T*>(a.normed) + row * a.cols + c, n, pack<T>(f));
    }
  }
  const uint32_t mine = magnitude8(v);
  const bool finite = all_finite(v);
  uint32_t top = block_max(mine);
  if (NORM) {  // a factor that is NaN, or infinite times zero, leaves no finite value: as for a block of zeros
    const float largest = __uint_as_float(top) * inv;
    top = largest >= 0.f ? min(__float_as_uint(largest), 0x7F7FFFFFu) : 0u;
  }
  const uint32_t e = scale_exponent(top);
  float factor = reciprocal_of(e);
  if (NORM) {
    if (inv * factor < __uint_as_float(0x7F800000u)) {
      factor *= inv;
    } else {  // a block of zeros or nearly so: the scale's reciprocal is 2^126, and 0 times infinity is no 0
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = mul2(v[i], make_float2(inv, inv));
    }
  }
  store8_e4m3<VEC>(a.q + row * a.cols + c, n, pack8(v, factor, finite));
  if (n > 0 && (threadIdx.x & 15) == 0) a.scale[row * blocks + c / kBlock] = (uint8_t)e;
}
template <typename T, bool VEC>
__device__ __forceinline__ void load_weight(const RowFp8& a, int c, float2 (&w)[4]) {
  if (a.weight_type == Type::kF32)
    unpack(load_raw<VEC>(static_cast<const float*>(a.weight) + c, a.cols - c), w);
  else
    unpack(load_raw<VEC>(static_cast<const T*>(a.weight) + c, a.cols - c), w);
}
__device__ __forceinline__ float warp_sum(float sum) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return sum;
}

// A CTA per row (or a warp, four to a CTA); everything that a row needs is on its way before the first sum.  VEC: all rows and
// the weight start on 16-byte boundaries and hold whole vectors.  (Where that is asked per vector, the two
// ways meet behind every load, and the loads go one by one.)
template <typename T, int V, bool NORM, bool VEC>
__global__ void __launch_bounds__(1024) row_fp8_kernel(const RowFp8 a) {
  allow_successor();
  wait_predecessors();
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const bool here = row < a.rows, has_residual = NORM && a.residual != nullptr;
  const T* x = static_cast<const T*>(a.x) + row * a.x_ld;
  const T* r = static_cast<const T*>(a.residual) + row * a.residual_ld;
  auto column = [&](int j) { return (int)(j * blockDim.x + threadIdx.x) * 8; };
  auto count = [&](int j) { return here ? a.cols - column(j) : 0; };
  Eight<T> rx[V], rr[V];
  float2 w[V][4], v[V][4];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    rx[j] = load_raw<VEC>(x + column(j), count(j));
    if (has_residual) rr[j] = load_raw<VEC>(r + column(j), count(j));
    if (NORM) load_weight<T, VEC>(a, column(j), w[j]);
  }
  float2 squares = make_float2(0.f, 0.f);
#pragma unroll
  for (int j = 0; j < V; ++j) {
    if (has_residual) {
      rx[j] = add(rx[j], rr[j]);
      store_raw<VEC>(static_cast<T*>(a.sum) + row * a.cols + column(j), count(j), rx[j]);
    }
    unpack(rx[j], v[j]);
    if (NORM) {
#pragma unroll
      for (int i = 0; i < 4; ++i) squares = fma2(v[j][i], v[j][i], squares);
    }
  }
  float inv = 1.f;
  if (NORM) {
    float sum = warp_sum(squares.x + squares.y);
    if (warps > 1) {  // one row per CTA
      __shared__ float part[32];
      if (lane == 0) part[warp] = sum;
      __syncthreads();
      sum = warp_sum(lane < warps ? part[lane] : 0.f);
    }
    inv = __frsqrt_rn(fmaf(sum, 1.f / (float)a.cols, a.eps));
  }
  const int blocks = (a.cols + kBlock - 1) / kBlock;
#pragma unroll
  for (int j = 0; j < V; ++j) finish<T, NORM, VEC>(a, v[j], w[j], inv, row, column(j), count(j), blocks);
}

// Many rows: a CTA goes through them, its threads holding V vectors of a row each, and loads the next row while it
// works on this one; the weight stays in registers.  With one row per CTA the instructions around the arithmetic (addresses,
// the sum over the CTA) were most of all, and issuing them the bound: 104 us for 8192 rows of 7168.
constexpr int kStreamVectors = 2;
constexpr int kStreamThreads = 448;  // per CTA, at most; two of them per SM leave a thread 72 registers
template <typename T, bool NORM>
__global__ void __launch_bounds__(kStreamThreads, 2) row_stream_fp8_kernel(const RowFp8 a) {
  constexpr int V = kStreamVectors;
  allow_successor();
  wait_predecessors();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const bool has_residual = NORM && a.residual != nullptr;
  const int blocks = (a.cols + kBlock - 1) / kBlock;
  const float share = 1.f / (float)a.cols;
  const int64_t step = (int64_t)gridDim.x * blockDim.y;
  int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  auto column = [&](int j) { return (int)(j * blockDim.x + threadIdx.x) * 8; };
  Eight<T> rx[V], rr[V], rw[V];
  auto fetch = [&]() {
    const T* x = static_cast<const T*>(a.x) + row * a.x_ld;
    const T* r = static_cast<const T*>(a.residual) + row * a.residual_ld;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int n = row < a.rows ? a.cols - column(j) : 0;
      rx[j] = load_raw<true>(x + column(j), n);
      if (has_residual) rr[j] = load_raw<true>(r + column(j), n);
    }
  };
  fetch();
  if (NORM) {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (a.weight_type != Type::kF32) rw[j] = load_raw<true>(static_cast<const T*>(a.weight) + column(j), a.cols - column(j));
  }
  for (int turn = 0; row - threadIdx.y < a.rows; turn ^= 1) {  // the CTA's rows stay together
    const int64_t here = row;
    auto count = [&](int j) { return here < a.rows ? a.cols - column(j) : 0; };
    float2 v[V][4], squares = make_float2(0.f, 0.f);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (has_residual) {
        rx[j] = add(rx[j], rr[j]);
        store_raw<true>(static_cast<T*>(a.sum) + here * a.cols + column(j), count(j), rx[j]);
      }
      unpack(rx[j], v[j]);
      if (NORM) {
#pragma unroll
        for (int i = 0; i < 4; ++i) squares = fma2(v[j][i], v[j][i], squares);
      }
    }
    row += step;
    fetch();
    float inv = 1.f;
    if (NORM) {
      float sum = warp_sum(squares.x + squares.y);
      if (warps > 1) {  // one row per CTA
        __shared__ float part[2][kStreamThreads / 32];
        if (lane == 0) part[turn][warp] = sum;
        __syncthreads();
        sum = warp_sum(lane < warps ? part[turn][lane] : 0.f);
      }
      inv = __frsqrt_rn(fmaf(sum, share, a.eps));
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float2 w[4];
      if (NORM && a.weight_type == Type::kF32)
        load_weight<T, true>(a, column(j), w);
      else if (NORM)
        unpack(rw[j], w);
      finish<T, NORM, true>(a, v[j], w, inv, here, column(j), count(j), blocks);
    }
  }
}

template <typename T, bool NORM, bool VEC>
cudaError_t launch_rows(const RowFp8& a, int n_sms, cudaStream_t stream) {
  const int vectors = (a.cols + 7) / 8;
  if constexpr (VEC) {
    constexpr int V = kStreamVectors;
    const int threads = (vectors + 32 * V - 1) / (32 * V) * 32;
    if (a.rows > 16 * n_sms && threads <= kStreamThreads) {
      const int per_cta = threads == 32 ? 4 : 1;
      int64_t grid = (a.rows + per_cta - 1) / per_cta;
      const int64_t most = (int64_t)n_sms * (2 * kStreamThreads / (threads * per_cta));
      if (grid > most) grid = most;
      auto kernel = row_stream_fp8_kernel<T, NORM>;
      return launch_after(kernel, dim3((unsigned)grid), dim3(threads, per_cta), 0, stream, a);
    }
  }
  // Else a CTA per row, as many threads as it has vectors: the chain of loads, sums and stores of a row
  // is all there is.
  const int v = vectors > 1024 ? 2 : 1;
  const int threads = (vectors + 32 * v - 1) / (32 * v) * 32;
  const int per_cta = threads == 32 ? 4 : 1;
  const dim3 block(threads, per_cta);
  const int64_t grid = (a.rows + per_cta - 1) / per_cta;
  if (threads > 1024 || grid > 0x7fffffff) return cudaErrorInvalidValue;
  auto kernel = v == 2 ? row_fp8_kernel<T, 2, NORM, VEC> : row_fp8_kernel<T, 1, NORM, VEC>;
  return launch_after(kernel, dim3((unsigned)grid), block, 0, stream, a);
}

// One CTA per 128 x 128 block, a row of it to 16 threads; weights are laid out once, so this is not
// tuned beyond reading and writing whole sectors.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) weight_fp8_kernel(const T* w, int64_t rows, int64_t cols, int64_t row_blocks,
                                                         int64_t col_blocks, uint8_t* q, uint8_t* scale) {
  allow_successor();
  wait_predecessors();
  const int64_t block = blockIdx.x;
  const int64_t cb = block % col_blocks, rb = block / col_blocks % row_blocks, m = block / col_blocks / row_blocks;
  const int64_t c = cb * kBlock + (threadIdx.x & 15) * 8;
  const int n = (int)max((int64_t)0, min((int64_t)8, cols - c));
  float2 v[8][4];
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int64_t r = rb * kBlock + j * 16 + (threadIdx.x >> 4);
    unpack(load_raw<VEC>(w + (m * rows + r) * cols + c, r < rows ? n : 0), v[j]);
    top = max(top, magnitude8(v[j]));
  }
  __shared__ uint32_t part[8];
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, part[i]);
  const uint32_t e = scale_exponent(top);
  const float reciprocal = reciprocal_of(e);
  if (threadIdx.x == 0) scale[block] = (uint8_t)e;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int64_t r = rb * kBlock + j * 16 + (threadIdx.x >> 4);
    if (r < rows && n > 0) store8_e4m3<VEC>(q + (m * rows + r) * cols + c, n, pack8(v[j], reciprocal, all_finite(v[j])));
  }
}

}  // namespace

namespace {
template <typename T>
cudaError_t launch_rows(const RowFp8& a, int n_sms, cudaStream_t stream) {
  auto whole = [&](const void* p, int64_t ld, size_t size) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (a.rows < 2 || ld * size % 16 == 0); };
  const bool vec = a.cols % 8 == 0 && whole(a.x, a.x_ld, sizeof(T)) && whole(a.residual, a.residual_ld, sizeof(T)) && whole(a.weight, 0, 1);
  if (a.weight) return vec ? launch_rows<T, true, true>(a, n_sms, stream) : launch_rows<T, true, false>(a, n_sms, stream);
  return vec ? launch_rows<T, false, true>(a, n_sms, stream) : launch_rows<T, false, false>(a, n_sms, stream);
}
template <typename T>
cudaError_t launch_weight(const void* w, int64_t blocks, int64_t rows, int64_t cols, uint8_t* q, uint8_t* scale, cudaStream_t stream) {
  const int64_t rb = (rows + kBlock - 1) / kBlock, cb = (cols + kBlock - 1) / kBlock;
  auto kernel = cols % 8 == 0 && (reinterpret_cast<uintptr_t>(w) & 15) == 0 ? weight_fp8_kernel<T, true> : weight_fp8_kernel<T, false>;
  return launch_after(kernel, dim3((unsigned)blocks), 256, 0, stream, static_cast<const T*>(w), rows, cols, rb, cb, q, scale);
}
}  // namespace

cudaError_t launch_row_fp8(const RowFp8& a, int n_sms, cudaStream_t stream) {
  if (a.rows < 0 || a.cols < 1 || a.cols > kMaxRowLength) return cudaErrorInvalidValue;
  if (a.rows == 0) return cudaSuccess;
  switch (a.type) {
    case Type::kF32: return launch_rows<float>(a, n_sms, stream);
    case Type::kBf16: return launch_rows<__nv_bfloat16>(a, n_sms, stream);
    default: return launch_rows<__half>(a, n_sms, stream);
  }
}

cudaError_t launch_weight_fp8(const void* w, Type type, int64_t matrices, int64_t rows, int64_t cols, uint8_t* q, uint8_t* scale,
                              cudaStream_t stream) {
  const int64_t blocks = matrices * ((rows + kBlock - 1) / kBlock) * ((cols + kBlock - 1) / kBlock);
  if (matrices < 0 || rows < 0 || cols < 0 || blocks > 0x7fffffff) return cudaErrorInvalidValue;
  if (blocks == 0) return cudaSuccess;
  switch (type) {
    case Type::kF32: return launch_weight<float>(w, blocks, rows, cols, q, scale, stream);
    case Type::kBf16: return launch_weight<__nv_bfloat16>(w, blocks, rows, cols, q, scale, stream);
    default: return launch_weight<__half>(w, blocks, rows, cols, q, scale, stream);
  }
}

}  // namespace ops
}  // namespace lplb

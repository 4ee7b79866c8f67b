// Rows to 8 bits, with the residual's addition and the root-mean-square norm in front.
//
//   h = round(x + r)            to x's type: the sum is an output, and what the next layer sees is normed
//   n = h * w / sqrt(mean(h^2) + eps)
//   s = 2^ceil(log2(max|n| / 448))   per block of 128,   q = e4m3(n / s)
//
// One pass: a row's values stay in registers between the sum of squares and the conversion, so x, r
// and w are read once and h, q and s written once.  Everything between is in 32 bits.
#include "ops_api.h"

#include "common.cuh"
#include "fp8.cuh"

namespace lplb {
namespace ops {
namespace {

using namespace fp8;

// A row belongs to blockDim.x threads (whole warps), every thread to V vectors of eight values that are
// blockDim.x vectors apart; 16 neighbouring lanes hold a block of 128.  Rows of one warp share a CTA.
template <typename T, int V, bool NORM>
__global__ void __launch_bounds__(1024) row_fp8_kernel(const RowFp8 a) {
  allow_successor();
  wait_predecessors();
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const bool here = row < a.rows;
  const T* x = static_cast<const T*>(a.x) + row * a.x_ld;
  const T* r = static_cast<const T*>(a.residual) + row * a.residual_ld;
  const bool x_vec = ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(a.residual ? r : x)) & 15) == 0;
  const bool out_vec = (a.cols & 7) == 0;
  float v[V][8];
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int c = (j * blockDim.x + threadIdx.x) * 8, n = here ? min(8, a.cols - c) : 0;
    load8(x + c, n >= 8 && x_vec, n, v[j]);
  }
  if (NORM && a.residual != nullptr) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = (j * blockDim.x + threadIdx.x) * 8, n = here ? min(8, a.cols - c) : 0;
      float f[8];
      load8(r + c, n >= 8 && x_vec, n, f);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[j][i] = to_float(from_float<T>(v[j][i] + f[i]));
      if (n > 0) store8(static_cast<T*>(a.sum) + row * a.cols + c, n == 8 && out_vec, n, v[j]);
    }
  }
  if (NORM) {
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) sum = fmaf(v[j][i], v[j][i], sum);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (warps > 1) {  // one row per CTA
      __shared__ float part[32];
      if (lane == 0) part[warp] = sum;
      __syncthreads();
      sum = lane < warps ? part[lane] : 0.f;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
  }
  const float inv = NORM ? __frsqrt_rn(sum / (float)a.cols + a.eps) : 1.f;
  const int blocks = (a.cols + kBlock - 1) / kBlock;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int c = (j * blockDim.x + threadIdx.x) * 8, n = here ? min(8, a.cols - c) : 0;
    if (NORM) {
      float w[8];
      const bool vec = n >= 8 && (reinterpret_cast<uintptr_t>(a.weight) & 15) == 0;
      if (a.weight_type == Type::kF32)
        load8(static_cast<const float*>(a.weight) + c, vec, n, w);
      else
        load8(static_cast<const T*>(a.weight) + c, vec, n, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[j][i] = v[j][i] * inv * w[i];
      if (a.normed != nullptr && n > 0) store8(static_cast<T*>(a.normed) + row * a.cols + c, n == 8 && out_vec, n, v[j]);
    }
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, magnitude(v[j][i]));
    const uint32_t e = scale_exponent(block_max(top));
    if (n > 0) {
      store8_e4m3(a.q + row * a.cols + c, n == 8 && out_vec, n, pack8(v[j], reciprocal_of(e)));
      if ((lane & 15) == 0) a.scale[row * blocks + c / kBlock] = (uint8_t)e;
    }
  }
}

template <typename T, bool NORM>
cudaError_t launch_rows(const RowFp8& a, int n_sms, cudaStream_t stream) {
  const int vectors = (a.cols + 7) / 8;
  // Vectors per thread: one where a row's threads are few or the rows leave SMs idle anyway (the chain
  // of one row's loads, sums and stores is all there is), four where many rows wait.
  const int v = vectors > 2048 || (vectors > 128 && a.rows > 4 * n_sms) ? 4 : vectors > 1024 ? 2 : 1;
  const int threads = (vectors + 32 * v - 1) / (32 * v) * 32;
  const int per_cta = threads == 32 ? 4 : 1;
  const dim3 block(threads, per_cta);
  const int64_t grid = (a.rows + per_cta - 1) / per_cta;
  if (threads > 1024 || grid > 0x7fffffff) return cudaErrorInvalidValue;
  if (v == 4) return launch_after(row_fp8_kernel<T, 4, NORM>, dim3((unsigned)grid), block, 0, stream, a);
  if (v == 2) return launch_after(row_fp8_kernel<T, 2, NORM>, dim3((unsigned)grid), block, 0, stream, a);
  return launch_after(row_fp8_kernel<T, 1, NORM>, dim3((unsigned)grid), block, 0, stream, a);
}

// One CTA per 128 x 128 block, a row of it to 16 threads; weights are laid out once, so this is not
// tuned beyond reading and writing whole sectors.
template <typename T>
__global__ void __launch_bounds__(256) weight_fp8_kernel(const T* __restrict__ w, int64_t rows, int64_t cols, int64_t row_blocks,
                                                         int64_t col_blocks, uint8_t* q, uint8_t* scale) {
  allow_successor();
  wait_predecessors();
  const int64_t block = blockIdx.x;
  const int64_t cb = block % col_blocks, rb = block / col_blocks % row_blocks, m = block / col_blocks / row_blocks;
  const int64_t c = cb * kBlock + (threadIdx.x & 15) * 8;
  const int n = (int)max((int64_t)0, min((int64_t)8, cols - c));
  const bool vec = n == 8 && (cols & 7) == 0 && (reinterpret_cast<uintptr_t>(w) & 15) == 0;
  float v[8][8];
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int64_t r = rb * kBlock + j * 16 + (threadIdx.x >> 4);
    load8(w + (m * rows + r) * cols + c, vec && r < rows, r < rows ? n : 0, v[j]);
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, magnitude(v[j][i]));
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
    if (r < rows && n > 0) store8_e4m3(q + (m * rows + r) * cols + c, n == 8 && (cols & 7) == 0, n, pack8(v[j], reciprocal));
  }
}

}  // namespace

cudaError_t launch_row_fp8(const RowFp8& a, int n_sms, cudaStream_t stream) {
  if (a.rows < 0 || a.cols < 1 || a.cols > kMaxRowLength) return cudaErrorInvalidValue;
  if (a.rows == 0) return cudaSuccess;
  switch (a.type) {
    case Type::kF32: return a.weight ? launch_rows<float, true>(a, n_sms, stream) : launch_rows<float, false>(a, n_sms, stream);
    case Type::kBf16:
      return a.weight ? launch_rows<__nv_bfloat16, true>(a, n_sms, stream) : launch_rows<__nv_bfloat16, false>(a, n_sms, stream);
    default: return a.weight ? launch_rows<__half, true>(a, n_sms, stream) : launch_rows<__half, false>(a, n_sms, stream);
  }
}

cudaError_t launch_weight_fp8(const void* w, Type type, int64_t matrices, int64_t rows, int64_t cols, uint8_t* q, uint8_t* scale,
                              cudaStream_t stream) {
  const int64_t rb = (rows + kBlock - 1) / kBlock, cb = (cols + kBlock - 1) / kBlock, blocks = matrices * rb * cb;
  if (matrices < 0 || rows < 0 || cols < 0 || blocks > 0x7fffffff) return cudaErrorInvalidValue;
  if (blocks == 0) return cudaSuccess;
  switch (type) {
    case Type::kF32:
      return launch_after(weight_fp8_kernel<float>, dim3((unsigned)blocks), 256, 0, stream, static_cast<const float*>(w), rows, cols, rb, cb, q, scale);
    case Type::kBf16:
      return launch_after(weight_fp8_kernel<__nv_bfloat16>, dim3((unsigned)blocks), 256, 0, stream, static_cast<const __nv_bfloat16*>(w),
                          rows, cols, rb, cb, q, scale);
    default:
      return launch_after(weight_fp8_kernel<__half>, dim3((unsigned)blocks), 256, 0, stream, static_cast<const __half*>(w), rows, cols, rb, cb, q,
                          scale);
  }
}

}  // namespace ops
}  // namespace lplb

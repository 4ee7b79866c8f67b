// The router's choice: the k largest logits of every token and their weights, and the logits' gradient.
//
//   s = softmax(l) or sigmoid(l)
//   chosen: the k largest l above -infinity, in descending order, ties to the lower expert; a NaN counts as largest
//   w_r = scale * s[chosen_r]                      or, renormalised, scale * s[chosen_r] / sum over r of s[chosen_r]
//
// Both scores rise with the logit, so the logits themselves are compared: nothing is decided by a rounded score.  The gradient, with
// d = dL/dw and A = sum over r of d_r w_r / scale:
//
//   softmax                dl_j = scale p_j (d_j [j chosen] - A)
//   softmax, renormalised  dl_j = w_j (d_j - A)                   for the chosen, 0 for the others
//   sigmoid                dl_j = scale d_j s_j (1 - s_j)
//   sigmoid, renormalised  dl_j = w_j (d_j - A) (1 - s_j)
//
// A warp has a token and holds its logits in registers, a lane every 32nd.  Logits become integers that compare as they do; a round of
// the choice is a warp reduction for the largest and one for the lowest expert that has it.  Bound by these dependent rounds.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "experts_api.h"

namespace lplb {
namespace ops {
namespace {

constexpr int kGateWarps = 4;
constexpr uint32_t kAll = 0xffffffffu;

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
__device__ __forceinline__ void narrow(float* p, float v) { *p = v; }
__device__ __forceinline__ void narrow(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void narrow(__half* p, float v) { *p = __float2half_rn(v); }

__device__ __forceinline__ float infinity() { return __uint_as_float(0x7F800000u); }
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {  // passes over NaN
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kAll, v, o));
  return v;
}

// An integer that compares as the logit does: 0 for -infinity, the largest for any NaN, the same for both zeros.
__device__ __forceinline__ uint32_t key_of(float v) {
  if (v != v) return kAll;
  if (v == -infinity()) return 0;
  const uint32_t b = __float_as_uint(v + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key); }

// 1 / (1 + e^-v), over e^min(most, 0) where that is given: the factor cancels in a renormalised weight, and the largest of a row
// of very small scores stays above one half.
__device__ __forceinline__ float sigmoid_over(float v, float most) {
  return expf(fminf(v, 0.f) - fminf(most, 0.f)) / (1.f + expf(-fabsf(v)));
}

// Score of this lane's choice, before the scale: `mine` is its logit (`there`: it has one), `most` the token's largest, `total` the
// softmax's sum.
__device__ __forceinline__ float score_of(const Gate& g, bool there, float mine, float most, float total) {
  if (g.sigmoid) {
    const float s = there ? sigmoid_over(mine, g.renormalize ? most : 0.f) : 0.f;
    return g.renormalize ? s / warp_sum(s) : s;
  }
  const float p = there ? expf(mine - most) : 0.f;
  return p / (g.renormalize ? warp_sum(p) : total);
}

template <typename T, int V>
__device__ __forceinline__ void load_logits(const Gate& g, int64_t token, int lane, float (&x)[V]) {
  const T* row = static_cast<const T*>(g.logits) + token * g.ld;
#pragma unroll
  for (int j = 0; j < V; ++j) x[j] = j * 32 + lane < g.experts ? widen(row[j * 32 + lane]) : -infinity();
}
template <int V>
__device__ __forceinline__ float softmax_sum(const float (&x)[V], float most) {
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < V; ++j) sum += expf(x[j] - most);
  return warp_sum(sum);
}

template <typename T, int V>
__global__ void __launch_bounds__(kGateWarps * 32) gate_kernel(const Gate g) {
  wait_predecessors();
  allow_successor();
  const int lane = threadIdx.x & 31;
  const int64_t token = (int64_t)blockIdx.x * kGateWarps + (threadIdx.x >> 5);
  if (token >= g.tokens) return;
  float x[V];
  load_logits<T, V>(g, token, lane, x);
  uint32_t key[V];
#pragma unroll
  for (int j = 0; j < V; ++j) key[j] = key_of(x[j]);
  uint32_t best = 0;
  int best_at = 0;  // this lane's largest, the lowest of equal ones
  auto look = [&] {
    best = key[0], best_at = 0;
#pragma unroll
    for (int j = 1; j < V; ++j)
      if (key[j] > best) best = key[j], best_at = j;
  };
  look();
  uint32_t largest = 0, mine = 0;
  int expert = -1;
  for (int r = 0; r < g.topk; ++r) {
    const uint32_t top = __reduce_max_sync(kAll, best);
    if (top == 0) break;
    if (r == 0) largest = top;
    const int candidate = best == top ? best_at * 32 + lane : INT32_MAX;
    const int winner = __reduce_min_sync(kAll, candidate);
    if (lane == r) mine = top, expert = winner;
    if (candidate == winner) {  // one lane's: the numbers differ
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (j == best_at) key[j] = 0;
      look();
    }
  }
  const float most = value_of(largest);
  const float total = !g.sigmoid && !g.renormalize && largest ? softmax_sum(x, most) : 1.f;
  const float score = score_of(g, expert >= 0, value_of(mine), most, total);
  if (lane < g.topk) {
    g.weights[token * g.topk + lane] = expert >= 0 ? g.scale * score : 0.f;
    g.idx[token * g.topk + lane] = expert;
  }
}

template <typename T, int V>
__global__ void __launch_bounds__(kGateWarps * 32) gate_backward_kernel(const Gate g) {
  wait_predecessors();
  allow_successor();
  const int lane = threadIdx.x & 31;
  const int64_t token = (int64_t)blockIdx.x * kGateWarps + (threadIdx.x >> 5);
  if (token >= g.tokens) return;
  const bool dense = !g.sigmoid && !g.renormalize;  // every logit has a gradient
  int expert = -1;
  float d = 0.f, mine = -infinity();
  if (lane < g.topk) {
    expert = (int)g.idx[token * g.topk + lane];
    if ((unsigned)expert < (unsigned)g.experts) {
      d = g.scale * g.dweights[token * g.topk + lane];
      mine = widen(static_cast<const T*>(g.logits)[token * g.ld + expert]);
    } else {
      expert = -1;
    }
  }
  float x[V];
  const float most = warp_max(mine);
  const bool any = __any_sync(kAll, expert >= 0);
  float total = 1.f;
  if (dense) {
    load_logits<T, V>(g, token, lane, x);
    if (any) total = softmax_sum(x, most);
  }
  const float score = score_of(g, expert >= 0, mine, most, total);
  const float along = g.sigmoid && !g.renormalize ? 0.f : warp_sum(expert >= 0 ? d * score : 0.f);
  float grad = score * (dense ? d : d - along);
  if (g.sigmoid) grad *= 1.f / (1.f + expf(mine));
  if (expert < 0) grad = 0.f;
#pragma unroll
  for (int j = 0; j < V; ++j) x[j] = dense && any ? -along * (expf(x[j] - most) / total) : 0.f;
  for (int r = 0; r < g.topk; ++r) {
    const int e = __shfl_sync(kAll, expert, r);
    const float more = __shfl_sync(kAll, grad, r);
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (j * 32 + lane == e) x[j] += more;
  }
  T* out = static_cast<T*>(g.dlogits) + token * g.experts;
#pragma unroll
  for (int j = 0; j < V; ++j)
    if (j * 32 + lane < g.experts) narrow(out + j * 32 + lane, x[j]);
}

template <typename T, int V>
cudaError_t launch(const Gate& g, bool backward, cudaStream_t stream) {
  auto kernel = backward ? gate_backward_kernel<T, V> : gate_kernel<T, V>;
  return launch_after(kernel, dim3((unsigned)((g.tokens + kGateWarps - 1) / kGateWarps)), dim3(kGateWarps * 32), 0, stream, g);
}
template <typename T>
cudaError_t launch(const Gate& g, bool backward, cudaStream_t stream) {
  if (g.experts <= 64) return launch<T, 2>(g, backward, stream);
  if (g.experts <= 128) return launch<T, 4>(g, backward, stream);
  if (g.experts <= 256) return launch<T, 8>(g, backward, stream);
  if (g.experts <= 512) return launch<T, 16>(g, backward, stream);
  return launch<T, 32>(g, backward, stream);
}
cudaError_t launch(const Gate& g, bool backward, cudaStream_t stream) {
  if (g.tokens < 0 || g.tokens > INT32_MAX || g.experts < 1 || g.experts > kGateMaxExperts || g.topk < 1 || g.topk > kGateMaxTopk ||
      g.topk > g.experts)
    return cudaErrorInvalidValue;
  if (g.tokens == 0) return cudaSuccess;
  switch (g.type) {
    case Type::kF32: return launch<float>(g, backward, stream);
    case Type::kBf16: return launch<__nv_bfloat16>(g, backward, stream);
    default: return launch<__half>(g, backward, stream);
  }
}

}  // namespace

cudaError_t launch_gate(const Gate& g, cudaStream_t stream) { return launch(g, false, stream); }
cudaError_t launch_gate_backward(const Gate& g, cudaStream_t stream) { return launch(g, true, stream); }

}  // namespace ops
}  // namespace lplb

// Launcher of the MoE layer for a few tokens.
#include "moe_few.cuh"

#include <atomic>

#include "tensor_map.h"

namespace lplb {
namespace ops {
namespace {

// The workspace's parts, one after the other on 256-byte boundaries.
struct Parts {
  size_t plan_words, slot, token, pair, ready, act, act_scale, q, q_scale, partial, product, total;
  int slots, rows, cols, ctas, counters;
  Parts(const MoeFew& m, int ctas_) : ctas(ctas_) {
    cols = (m.tokens + 15) / 16 * 16;
    rows = m.tokens * m.topk;
    slots = m.experts < rows ? m.experts : rows;
    counters = slots + slots * (m.inter / 128) + 1;
    const size_t value = m.w13_scale ? 1 : 2;
    size_t at = 0;
    auto take = [&](size_t bytes) {
      const size_t here = at;
      at += (bytes + 255) / 256 * 256;
      return here;
    };
    plan_words = take(8);
    slot = take((size_t)slots * sizeof(int2));
    token = take((size_t)rows + 4);
    pair = take((size_t)rows * sizeof(int2));
    ready = take((size_t)counters * 4);
    act = take((size_t)rows * m.inter * value);
    act_scale = take((size_t)rows * (m.inter / 128));
    const bool convert = m.w13_scale && !m.x_scale;
    q = take(convert ? (size_t)m.tokens * m.hidden : 0);
    q_scale = take(convert ? (size_t)m.tokens * (m.hidden / 128) : 0);
    // tiles in parts: no more parts than CTAs
    partial = take((size_t)ctas * (2 * cols * 128) * 4);
    product = take((size_t)kFewPieces * rows * m.hidden * 4);
    total = at;
  }
};

template <bool FP8>
cudaError_t launch(const FewMoeArgs& a, const CUtensorMap (&maps)[4], int n_sms, int device, cudaStream_t stream) {
  auto kernel = moe_few_kernel<FP8>;
  static std::atomic<bool> prepared[kMaxDevices];
  if (!prepared[device].load(std::memory_order_relaxed)) {
    const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewMoeSmem);
    if (err != cudaSuccess) return err;
    prepared[device].store(true, std::memory_order_relaxed);
  }
  return launch_after(kernel, dim3(n_sms), dim3(kFewMoeThreads), kFewMoeSmem, stream, maps[0], maps[1], maps[2], maps[3], a);
}

bool map_of(CUtensorMap* map, bool fp8, const void* base, uint64_t rows, uint64_t cols, uint64_t ld, uint32_t box_rows) {
  const uint64_t value = fp8 ? 1 : 2;
  const cuuint64_t dims[2] = {cols, rows}, strides[1] = {ld * value};
  const cuuint32_t box[2] = {(cuuint32_t)(kKBytes / value), box_rows};
  return encode_tensor_map(map, fp8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, base, 2, dims, strides, box) == 0;
}

}  // namespace

cudaError_t moe_few_workspace(const MoeFew& m, int device, size_t* bytes) {
  int n = 0;
  const cudaError_t err = multiprocessors(device, &n);
  if (err == cudaSuccess) *bytes = Parts(m, n).total;
  return err;
}

cudaError_t launch_moe_few(const MoeFew& m, int device, cudaStream_t stream) {
  const bool fp8 = m.w13_scale != nullptr;
  if (m.tokens < 0 || m.tokens > kMoeFewMaxTokens || m.topk < 1 || m.topk > kMoeFewMaxTopk || m.experts < 1 || m.experts > kMoeFewMaxExperts ||
      m.hidden < 256 || m.hidden % 256 || m.inter < 128 || m.inter % 128 || device < 0 || device >= kMaxDevices ||
      (int64_t)m.experts * 2 * m.inter > INT32_MAX || (int64_t)m.experts * m.hidden > INT32_MAX)
    return cudaErrorInvalidValue;
  if (m.tokens == 0) return cudaSuccess;
  int n_sms = 0;
  cudaError_t err = multiprocessors(device, &n_sms);
  if (err != cudaSuccess) return err;
  const Parts at(m, n_sms);
  char* ws = static_cast<char*>(m.workspace);
  MoeFewPlan plan;
  plan.slots = reinterpret_cast<int*>(ws + at.plan_words);
  plan.ticket = plan.slots + 1;
  plan.slot = reinterpret_cast<int2*>(ws + at.slot);
  plan.token = reinterpret_cast<uint8_t*>(ws + at.token);
  plan.pair = reinterpret_cast<int2*>(ws + at.pair);
  plan.ready = reinterpret_cast<int*>(ws + at.ready);
  plan.tile_parts = plan.ready + at.slots;
  plan.products = plan.tile_parts + (size_t)at.slots * (m.inter / 128);

  FewPlanArgs p{};
  p.plan = plan;
  p.idx = m.idx;
  p.weight = m.weight;
  p.is64 = m.idx_is64;
  p.tokens = m.tokens;
  p.topk = m.topk;
  p.experts = m.experts;
  p.counters = at.counters;
  const bool convert = fp8 && m.x_scale == nullptr;
  const void* x = m.x;
  int64_t x_ld = m.x_ld;
  FewMoeArgs a{};
  a.x_scale = m.x_scale;
  a.x_scale_ld = m.x_scale_ld;
  if (convert) {
    p.x = static_cast<const __nv_bfloat16*>(m.x);
    p.x_ld = m.x_ld;
    p.q = reinterpret_cast<uint8_t*>(ws + at.q);
    p.scale = reinterpret_cast<uint8_t*>(ws + at.q_scale);
    p.hidden = m.hidden;
    x = p.q;
    x_ld = m.hidden;
    a.x_scale = p.scale;
    a.x_scale_ld = m.hidden / 128;
  }
  a.plan = plan;
  a.w13_scale = m.w13_scale;
  a.w2_scale = m.w2_scale;
  a.act = ws + at.act;
  a.act_scale = reinterpret_cast<uint8_t*>(ws + at.act_scale);
  a.partial = reinterpret_cast<float*>(ws + at.partial);
  a.out = static_cast<__nv_bfloat16*>(m.out);
  a.product = reinterpret_cast<float*>(ws + at.product);
  a.tokens = m.tokens;
  a.topk = m.topk;
  a.cols = at.cols;
  a.hidden = m.hidden;
  a.inter = m.inter;
  const int per = fp8 ? 128 : 64;
  a.kb1 = m.hidden / per;
  a.kb2 = m.inter / per;
  a.ctas = at.ctas;
  a.slots = at.slots;
  a.x_words = a.x_scale_ld % 4 == 0 && (reinterpret_cast<uintptr_t>(a.x_scale) & 3) == 0;
  a.w_words = ((reinterpret_cast<uintptr_t>(a.w13_scale) | reinterpret_cast<uintptr_t>(a.w2_scale)) & 3) == 0;
  a.budget_ns = wait_budget_ns();
  a.error = m.status;
  if (a.error == nullptr && (err = ops_error_word(device, &a.error)) != cudaSuccess) return err;
  CUtensorMap maps[4];
  if (!map_of(&maps[0], fp8, m.w13, (uint64_t)m.experts * 2 * m.inter, m.hidden, m.hidden, kFewTileRows) ||
      !map_of(&maps[1], fp8, m.w2, (uint64_t)m.experts * m.hidden, m.inter, m.inter, kFewTileRows) ||
      !map_of(&maps[2], fp8, x, m.tokens, m.hidden, x_ld, 1) || !map_of(&maps[3], fp8, a.act, at.rows, m.inter, m.inter, 16))
    return cudaErrorInvalidValue;
  auto kernel = moe_few_plan_kernel;
  err = launch_after(kernel, dim3(1 + (convert ? m.tokens : 0)), dim3(kFewPlanThreads), 0, stream, p);
  if (err != cudaSuccess) return err;
  return fp8 ? launch<true>(a, maps, n_sms, device, stream) : launch<false>(a, maps, n_sms, device, stream);
}

}  // namespace ops
}  // namespace lplb

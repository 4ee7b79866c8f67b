// Python binding of the 8-bit serving operators: checks of the arguments, outputs, launches on the
// current stream of the arguments' device.  The reference has no operators of this kind.
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <pybind11/pybind11.h>
#include <pybind11/stl.h>
#include <torch/extension.h>

#include <optional>
#include <stdexcept>
#include <string>

#include "ops_api.h"

namespace py = pybind11;

namespace {

using torch::Tensor;
using OptTensor = std::optional<Tensor>;

// A refused argument is a ValueError, a failed launch a RuntimeError.  Messages are put together from strings: a
// number written to an ostringstream ends the process where the compiler's C++ library is newer than the one that
// is loaded.
#define OPS_CHECK(cond, msg)                                                       \
  do {                                                                             \
    if (!(cond)) throw std::invalid_argument(std::string("lplb_b200.ops.") + msg); \
  } while (0)

#define OPS_CUDA(expr)                                                                                            \
  do {                                                                                                            \
    cudaError_t err_ = (expr);                                                                                    \
    if (err_ != cudaSuccess)                                                                                      \
      throw std::runtime_error(std::string("lplb_b200.ops: " #expr " failed: ") + cudaGetErrorName(err_) + ": " + \
                               cudaGetErrorString(err_));                                                         \
  } while (0)

std::string text(int64_t n) { return std::to_string(n); }
std::string text(at::ScalarType type) { return c10::toString(type); }

constexpr int64_t kBlock = 128;
int64_t blocks_of(int64_t n) { return (n + kBlock - 1) / kBlock; }

lplb::ops::Type type_of(const Tensor& t, const char* who) {
  switch (t.scalar_type()) {
    case torch::kFloat32: return lplb::ops::Type::kF32;
    case torch::kBFloat16: return lplb::ops::Type::kBf16;
    case torch::kFloat16: return lplb::ops::Type::kF16;
    default: OPS_CHECK(false, who + std::string(" must be float32, bfloat16 or float16, not ") + text(t.scalar_type()));
  }
  return lplb::ops::Type::kF32;
}

void check_no_grad(const Tensor& t, const char* who) {
  OPS_CHECK(!(t.requires_grad() && at::GradMode::is_enabled()), who + std::string(" requires a gradient: these operators have no backward pass (use torch.no_grad())"));
}

int sm_count(int device) {
  int n = 0;
  OPS_CUDA(lplb::ops::multiprocessors(device, &n));
  return n;
}

cudaStream_t stream_of(int device) { return c10::cuda::getCurrentCUDAStream(device).stream(); }

// Rows of the last dimension as one matrix, without a copy wherever the strides allow it.
Tensor as_rows(const Tensor& t) { return t.dim() == 2 ? t : t.reshape({-1, t.size(-1)}); }

// An output on x's device, without the dispatcher's microsecond.
Tensor make(at::IntArrayRef sizes, at::ScalarType type, const Tensor& x) { return at::detail::empty_cuda(sizes, type, x.device(), std::nullopt); }

uint8_t* bytes(const Tensor& t) { return static_cast<uint8_t*>(t.data_ptr()); }

std::vector<int64_t> with_last(const Tensor& t, int64_t last) {
  auto shape = t.sizes().vec();
  shape.back() = last;
  return shape;
}

struct RowsOut {
  Tensor q, scale;
};
RowsOut make_rows(const Tensor& x) {
  const int64_t cols = x.size(-1);
  return {make(x.sizes(), torch::kFloat8_e4m3fn, x), make(with_last(x, blocks_of(cols)), torch::kFloat8_e8m0fnu, x)};
}

void check_rows(const Tensor& x, const char* who) {
  OPS_CHECK(x.is_cuda(), who + std::string(" must be a CUDA tensor"));
  OPS_CHECK(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= lplb::ops::kMaxRowLength,
            who + std::string(" must have rows of 1 to ") + text(lplb::ops::kMaxRowLength) + " values");
  OPS_CHECK(x.stride(-1) == 1 || x.size(-1) == 1 || x.numel() == 0, who + std::string(" must have the values of a row next to one another"));
  check_no_grad(x, who);
}

lplb::ops::RowFp8 row_args(const Tensor& x, const RowsOut& out, const char* who) {
  lplb::ops::RowFp8 a{};
  a.x = x.data_ptr();
  a.x_ld = x.stride(0);
  a.rows = x.size(0);
  a.cols = (int)x.size(1);
  a.q = bytes(out.q);
  a.scale = bytes(out.scale);
  a.type = type_of(x, who);
  return a;
}

py::tuple quantize_fp8(const Tensor& x) {
  check_rows(x, "quantize_fp8: x");
  c10::cuda::CUDAGuard guard(x.device());
  const auto out = make_rows(x);
  const Tensor rows = as_rows(x);
  OPS_CUDA(lplb::ops::launch_row_fp8(row_args(rows, out, "quantize_fp8: x"), sm_count(x.get_device()), stream_of(x.get_device())));
  return py::make_tuple(out.q, out.scale);
}

py::tuple rms_norm_fp8(const Tensor& x, const Tensor& weight, const OptTensor& residual, double eps, bool return_normed) {
  check_rows(x, "rms_norm_fp8: x");
  check_no_grad(weight, "rms_norm_fp8: weight");
  OPS_CHECK(weight.is_cuda() && weight.device() == x.device() && weight.dim() == 1 && weight.size(0) == x.size(-1) && weight.is_contiguous(),
            "rms_norm_fp8: weight must be contiguous, on x's device, one value for each of a row");
  OPS_CHECK(weight.scalar_type() == x.scalar_type() || weight.scalar_type() == torch::kFloat32, "rms_norm_fp8: weight must be float32 or of x's type");
  OPS_CHECK(eps >= 0, "rms_norm_fp8: eps must not be negative");
  c10::cuda::CUDAGuard guard(x.device());
  const Tensor rows = as_rows(x);
  const auto out = make_rows(x);
  auto a = row_args(rows, out, "rms_norm_fp8: x");
  a.weight = weight.data_ptr();
  a.weight_type = type_of(weight, "rms_norm_fp8: weight");
  a.eps = (float)eps;
  Tensor sum = x, normed, other;
  if (residual) {
    check_rows(*residual, "rms_norm_fp8: residual");
    OPS_CHECK(residual->device() == x.device() && residual->sizes() == x.sizes() && residual->scalar_type() == x.scalar_type(),
              "rms_norm_fp8: residual must have x's shape, type and device");
    other = as_rows(*residual);
    sum = make(x.sizes(), x.scalar_type(), x);
    a.residual = other.data_ptr();
    a.residual_ld = other.stride(0);
    a.sum = sum.data_ptr();
  }
  if (return_normed) {
    normed = make(x.sizes(), x.scalar_type(), x);
    a.normed = normed.data_ptr();
  }
  OPS_CUDA(lplb::ops::launch_row_fp8(a, sm_count(x.get_device()), stream_of(x.get_device())));
  if (return_normed) return py::make_tuple(out.q, out.scale, sum, normed);
  return py::make_tuple(out.q, out.scale, sum);
}

py::tuple quantize_weight_fp8(const Tensor& w) {
  OPS_CHECK(w.is_cuda() && (w.dim() == 2 || w.dim() == 3) && w.is_contiguous(), "quantize_weight_fp8: w must be a contiguous CUDA tensor [rows, cols] or [matrices, rows, cols]");
  check_no_grad(w, "quantize_weight_fp8: w");
  const auto type = type_of(w, "quantize_weight_fp8: w");
  c10::cuda::CUDAGuard guard(w.device());
  const int64_t matrices = w.dim() == 3 ? w.size(0) : 1, rows = w.size(-2), cols = w.size(-1);
  auto shape = w.sizes().vec();
  shape[shape.size() - 2] = blocks_of(rows);
  shape.back() = blocks_of(cols);
  auto q = make(w.sizes(), torch::kFloat8_e4m3fn, w);
  auto scale = make(shape, torch::kFloat8_e8m0fnu, w);
  OPS_CUDA(lplb::ops::launch_weight_fp8(w.data_ptr(), type, matrices, rows, cols, bytes(q), bytes(scale), stream_of(w.get_device())));
  return py::make_tuple(q, scale);
}

// Where a call's errors go, if not to the device's word.
int* status_of(const OptTensor& status, const at::Device& device, const char* who) {
  if (!status) return nullptr;
  OPS_CHECK(status->device() == device && status->scalar_type() == torch::kInt32 && status->numel() >= 1,
            who + std::string(": status must be int32 on the arguments' device"));
  return status->data_ptr<int>();
}

Tensor matmul_fp8(const Tensor& a, const Tensor& a_scale, const Tensor& b, const Tensor& b_scale, const OptTensor& rows, const OptTensor& out,
                  bool out_f32, const OptTensor& status) {
  const auto device = a.device();
  OPS_CHECK(a.is_cuda() && a.dim() == 2 && a.scalar_type() == torch::kFloat8_e4m3fn, "matmul_fp8: a must be a CUDA tensor [rows, k] of float8_e4m3fn");
  const int64_t lead = rows ? 1 : 0;  // dimensions in front of a matrix
  OPS_CHECK(b.device() == device && b.dim() == 2 + lead && b.scalar_type() == torch::kFloat8_e4m3fn,
            "matmul_fp8: b must be [n, k] (with rows: [groups, n, k]) of float8_e4m3fn on a's device");
  const int64_t m = a.size(0), k = a.size(1), n = b.size(-2), kb = blocks_of(k), groups = rows ? b.size(0) : 1;
  OPS_CHECK(groups >= 1 && groups <= lplb::ops::kMaxGroups, "matmul_fp8: 1 to " + text(lplb::ops::kMaxGroups) + " groups");
  OPS_CHECK(!rows || (rows->device() == device && rows->scalar_type() == torch::kInt32 && rows->dim() == 1 && rows->size(0) == groups && rows->is_contiguous()),
            "matmul_fp8: rows must be contiguous int32, one number for each matrix of b, on a's device");
  OPS_CHECK(m <= lplb::ops::kMaxRows && groups * n <= lplb::ops::kMaxRows,
            "matmul_fp8: at most " + text(lplb::ops::kMaxRows) + " rows of a, and of all matrices of b together");
  OPS_CHECK(k >= 16 && k % 16 == 0 && b.size(-1) == k, "matmul_fp8: a and b must have the same k, a multiple of 16");
  OPS_CHECK(n >= 1 && n < (1 << 28), "matmul_fp8: b has no rows, or too many");
  OPS_CHECK(a.stride(1) == 1 && (m < 2 || (a.stride(0) % 16 == 0 && a.stride(0) >= k)) && reinterpret_cast<uintptr_t>(a.data_ptr()) % 16 == 0,
            "matmul_fp8: rows of a must be contiguous, apart from one another and start on 16-byte boundaries");
  OPS_CHECK(b.is_contiguous() && reinterpret_cast<uintptr_t>(b.data_ptr()) % 16 == 0, "matmul_fp8: b must be contiguous and start on a 16-byte boundary");
  OPS_CHECK(a_scale.device() == device && a_scale.scalar_type() == torch::kFloat8_e8m0fnu && a_scale.dim() == 2 && a_scale.size(0) == m &&
                a_scale.size(1) == kb && (a_scale.stride(1) == 1 || kb == 1),
            "matmul_fp8: a_scale must be [rows, ceil(k / 128)] of float8_e8m0fnu on a's device, rows contiguous");
  OPS_CHECK(b_scale.device() == device && b_scale.scalar_type() == torch::kFloat8_e8m0fnu && b_scale.is_contiguous() &&
                b_scale.dim() == 2 + lead && (!rows || b_scale.size(0) == groups) && b_scale.size(-2) == blocks_of(n) && b_scale.size(-1) == kb,
            "matmul_fp8: b_scale must be contiguous [ceil(n / 128), ceil(k / 128)] (with rows: for every group) of float8_e8m0fnu on a's device");
  check_no_grad(a, "matmul_fp8: a");
  check_no_grad(b, "matmul_fp8: b");
  c10::cuda::CUDAGuard guard(device);
  const auto type = out_f32 ? torch::kFloat32 : torch::kBFloat16;
  Tensor result;
  if (out) {
    OPS_CHECK(out->device() == device && out->scalar_type() == type && out->dim() == 2 && out->size(0) == m && out->size(1) == n &&
                  (out->stride(1) == 1 || n == 1) && (m < 2 || out->stride(0) >= n),
              "matmul_fp8: out must be [rows, n] of the output type on a's device, rows contiguous and apart from one another");
    check_no_grad(*out, "matmul_fp8: out");
    result = *out;
    // what autograd has saved of `out` is no longer what it was
    if (!result.is_inference()) result.unsafeGetTensorImpl()->bump_version();
  } else {
    result = make({m, n}, type, a);
  }
  lplb::ops::Product p{};
  p.a = a.data_ptr();
  p.b = b.data_ptr();
  p.a_scale = bytes(a_scale);
  p.b_scale = bytes(b_scale);
  p.out = result.data_ptr();
  p.m = m;
  p.n = n;
  p.k = k;
  p.a_ld = m < 2 ? k : a.stride(0);
  p.rows = rows ? rows->data_ptr<int>() : nullptr;
  p.groups = (int)groups;
  p.a_scale_ld = m < 2 ? kb : a_scale.stride(0);
  p.out_ld = result.stride(0);
  p.out_f32 = out_f32;
  p.status = status_of(status, device, "matmul_fp8");
  OPS_CUDA(lplb::ops::launch_matmul_fp8(p, a.get_device(), stream_of(a.get_device())));
  return result;
}

Tensor moe_few_tokens(const Tensor& x, const Tensor& idx, const Tensor& weights, const Tensor& w13, const Tensor& w2, const OptTensor& x_scale,
                      const OptTensor& w13_scale, const OptTensor& w2_scale, const OptTensor& status) {
  const auto device = x.device();
  const bool fp8 = w13_scale.has_value();
  OPS_CHECK(x.is_cuda() && x.dim() == 2, "moe_few_tokens: x must be a CUDA tensor [tokens, hidden]");
  const int64_t tokens = x.size(0), hidden = x.size(1);
  OPS_CHECK(tokens <= lplb::ops::kMoeFewMaxTokens, "moe_few_tokens: at most " + text(lplb::ops::kMoeFewMaxTokens) + " tokens, not " + text(tokens));
  OPS_CHECK(fp8 == w2_scale.has_value(), "moe_few_tokens: w13_scale and w2_scale come together");
  OPS_CHECK(fp8 || !x_scale, "moe_few_tokens: x_scale needs weights in 8 bits");
  const auto wtype = fp8 ? torch::kFloat8_e4m3fn : torch::kBFloat16;
  OPS_CHECK(w13.device() == device && w13.dim() == 3 && w13.scalar_type() == wtype && w13.is_contiguous() && w2.device() == device && w2.dim() == 3 &&
                w2.scalar_type() == wtype && w2.is_contiguous(),
            "moe_few_tokens: w13 and w2 must be contiguous, on x's device, " + text(wtype));
  const int64_t experts = w13.size(0), inter = w13.size(1) / 2;
  OPS_CHECK(experts >= 1 && experts <= lplb::ops::kMoeFewMaxExperts, "moe_few_tokens: 1 to " + text(lplb::ops::kMoeFewMaxExperts) + " experts");
  OPS_CHECK(hidden >= 256 && hidden % 256 == 0 && inter >= 128 && inter % 128 == 0 && hidden <= lplb::ops::kMoeFewMaxHidden &&
                inter <= lplb::ops::kMoeFewMaxInter,
            "moe_few_tokens: hidden must be a multiple of 256 (up to " + text(lplb::ops::kMoeFewMaxHidden) + "), inter of 128 (up to " +
                text(lplb::ops::kMoeFewMaxInter) + ")");
  OPS_CHECK(w13.size(1) == 2 * inter && w13.size(2) == hidden && w2.size(0) == experts && w2.size(1) == hidden && w2.size(2) == inter,
            "moe_few_tokens: w13 must be [experts, 2 * inter, hidden], w2 [experts, hidden, inter]");
  OPS_CHECK(experts * 2 * inter <= INT32_MAX && experts * hidden <= INT32_MAX, "moe_few_tokens: more than 2^31 weight rows");
  const auto xtype = x_scale ? torch::kFloat8_e4m3fn : torch::kBFloat16;
  const int64_t xsize = x_scale ? 1 : 2;
  OPS_CHECK(x.scalar_type() == xtype, "moe_few_tokens: x must be bfloat16, or float8_e4m3fn with x_scale");
  OPS_CHECK(x.stride(1) == 1 && (tokens < 2 || (x.stride(0) * xsize % 16 == 0 && x.stride(0) >= hidden)) &&
                reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0,
            "moe_few_tokens: rows of x must be contiguous, apart from one another and start on 16-byte boundaries");
  for (const Tensor* w : {&w13, &w2})
    OPS_CHECK(reinterpret_cast<uintptr_t>(w->data_ptr()) % 16 == 0, "moe_few_tokens: weights must start on a 16-byte boundary");
  OPS_CHECK(idx.device() == device && idx.dim() == 2 && idx.size(0) == tokens && (idx.scalar_type() == torch::kInt64 || idx.scalar_type() == torch::kInt32),
            "moe_few_tokens: idx must be [tokens, topk] of int64 or int32 on x's device");
  const int64_t topk = idx.size(1);
  OPS_CHECK(topk >= 1 && topk <= lplb::ops::kMoeFewMaxTopk, "moe_few_tokens: 1 to " + text(lplb::ops::kMoeFewMaxTopk) + " choices per token");
  OPS_CHECK(weights.device() == device && weights.sizes() == idx.sizes() && weights.is_floating_point(),
            "moe_few_tokens: weights must be floating point, of idx's shape, on x's device");
  auto scales_ok = [&](const Tensor& s, const Tensor& w) {
    return s.device() == device && s.scalar_type() == torch::kFloat8_e8m0fnu && s.is_contiguous() && s.dim() == 3 && s.size(0) == w.size(0) &&
           s.size(1) == w.size(1) / kBlock && s.size(2) == w.size(2) / kBlock;
  };
  OPS_CHECK(!fp8 || (scales_ok(*w13_scale, w13) && scales_ok(*w2_scale, w2)),
            "moe_few_tokens: scales of the weights must be contiguous [experts, rows / 128, cols / 128] of float8_e8m0fnu on x's device");
  OPS_CHECK(!x_scale || (x_scale->device() == device && x_scale->scalar_type() == torch::kFloat8_e8m0fnu && x_scale->dim() == 2 &&
                         x_scale->size(0) == tokens && x_scale->size(1) == hidden / kBlock && x_scale->stride(1) == 1),
            "moe_few_tokens: x_scale must be [tokens, hidden / 128] of float8_e8m0fnu on x's device, rows contiguous");
  check_no_grad(x, "moe_few_tokens: x");
  check_no_grad(weights, "moe_few_tokens: weights");
  check_no_grad(w13, "moe_few_tokens: w13");
  check_no_grad(w2, "moe_few_tokens: w2");
  c10::cuda::CUDAGuard guard(device);
  const int index = x.get_device();
  auto out = make({tokens, hidden}, torch::kBFloat16, x);
  if (tokens == 0) return out;
  const Tensor ids = idx.is_contiguous() ? idx : idx.contiguous();
  const Tensor gate = weights.scalar_type() == torch::kFloat32 && weights.is_contiguous() ? weights : weights.to(torch::kFloat32).contiguous();
  lplb::ops::MoeFew m{};
  m.x = x.data_ptr();
  m.x_scale = x_scale ? bytes(*x_scale) : nullptr;
  m.idx = ids.data_ptr();
  m.weight = gate.data_ptr<float>();
  m.w13 = w13.data_ptr();
  m.w2 = w2.data_ptr();
  m.w13_scale = fp8 ? bytes(*w13_scale) : nullptr;
  m.w2_scale = fp8 ? bytes(*w2_scale) : nullptr;
  m.out = out.data_ptr();
  m.x_ld = tokens < 2 ? hidden : x.stride(0);
  m.x_scale_ld = x_scale ? (tokens < 2 ? hidden / kBlock : x_scale->stride(0)) : 0;
  m.idx_is64 = ids.scalar_type() == torch::kInt64;
  m.tokens = (int)tokens;
  m.topk = (int)topk;
  m.experts = (int)experts;
  m.hidden = (int)hidden;
  m.inter = (int)inter;
  m.status = status_of(status, device, "moe_few_tokens");
  // a workspace of this call alone: calls on two streams, or two captured graphs, share nothing
  size_t workspace_bytes = 0;
  OPS_CUDA(lplb::ops::moe_few_workspace(m, index, &workspace_bytes));
  auto workspace = make({(int64_t)workspace_bytes}, torch::kUInt8, x);
  m.workspace = workspace.data_ptr();
  OPS_CUDA(lplb::ops::launch_moe_few(m, index, stream_of(index)));
  return out;
}

int ops_error(int device, bool clear) {
  c10::cuda::CUDAGuard guard(device);
  int code = 0;
  OPS_CUDA(lplb::ops::read_ops_error(&code, clear));
  return code;
}

}  // namespace

void bind_ops(py::module_& m) {
  m.def("quantize_fp8", &quantize_fp8);
  m.def("quantize_weight_fp8", &quantize_weight_fp8);
  m.def("rms_norm_fp8", &rms_norm_fp8);
  m.def("matmul_fp8", &matmul_fp8);
  m.def("moe_few_tokens", &moe_few_tokens);
  m.def("ops_error", &ops_error);
  m.def("set_ops_timeout_us", [](double us) {
    OPS_CHECK(us >= 0 && us <= 1e9, "set_ops_timeout_us: between 0 and 1e9");
    lplb::ops::set_wait_budget_ns((unsigned long long)(us * 1e3));
  });
  m.attr("MOE_FEW_MAX_TOKENS") = lplb::ops::kMoeFewMaxTokens;
  m.attr("MOE_FEW_MAX_TOPK") = lplb::ops::kMoeFewMaxTopk;
  m.attr("MOE_FEW_MAX_EXPERTS") = lplb::ops::kMoeFewMaxExperts;
  m.attr("MOE_FEW_MAX_HIDDEN") = lplb::ops::kMoeFewMaxHidden;
  m.attr("MOE_FEW_MAX_INTER") = lplb::ops::kMoeFewMaxInter;
  m.attr("MAX_ROW_LENGTH") = lplb::ops::kMaxRowLength;
}

// What the operators' Python bindings share: refusals, failed launches, streams and outputs.
#pragma once

#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
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

inline std::string text(int64_t n) { return std::to_string(n); }
inline std::string text(at::ScalarType type) { return c10::toString(type); }

inline lplb::ops::Type type_of(const Tensor& t, const char* who) {
  switch (t.scalar_type()) {
    case torch::kFloat32: return lplb::ops::Type::kF32;
    case torch::kBFloat16: return lplb::ops::Type::kBf16;
    case torch::kFloat16: return lplb::ops::Type::kF16;
    default: OPS_CHECK(false, who + std::string(" must be float32, bfloat16 or float16, not ") + text(t.scalar_type()));
  }
  return lplb::ops::Type::kF32;
}

// A dual tensor of forward-mode differentiation goes through a kernel without its tangent: the derivative would be zero, with no error.
inline void check_no_tangent(const Tensor& t, const char* who) {
  OPS_CHECK(!t.defined() || !t._fw_grad(0).defined() || !c10::AutogradState::get_tls_state().get_fw_grad_mode(),
            who + std::string(" has a forward-mode tangent: these operators are differentiated backwards alone"));
}
inline void check_no_grad(const Tensor& t, const char* who) {
  check_no_tangent(t, who);
  OPS_CHECK(!(t.requires_grad() && at::GradMode::is_enabled()), who + std::string(" requires a gradient: these operators have no backward pass (use torch.no_grad())"));
}

// A lazily conjugated or negated view (z.conj(), z.conj().imag) stands for other values than its memory holds: what a kernel reads is written
// out first.  A recorded call does this before it is recorded, so that the gradient goes back through it.
inline Tensor as_stored(const Tensor& t) { return t.defined() && (t.is_conj() || t.is_neg()) ? t.resolve_conj().resolve_neg() : t; }
inline OptTensor as_stored(const OptTensor& t) { return t ? OptTensor(as_stored(*t)) : std::nullopt; }

// Whole numbers that a kernel reads one after the other, as an order's and a call's counts are.
inline Tensor in_a_row(const Tensor& t) { return t.is_contiguous() ? t : t.contiguous(); }

inline int sm_count(int device) {
  int n = 0;
  OPS_CUDA(lplb::ops::multiprocessors(device, &n));
  return n;
}

inline cudaStream_t stream_of(int device) { return c10::cuda::getCurrentCUDAStream(device).stream(); }

// Rows of the last dimension as one matrix, without a copy wherever the strides allow it.
inline Tensor as_rows(const Tensor& t) { return t.dim() == 2 ? t : t.reshape({-1, t.size(-1)}); }

// An output on x's device, without the dispatcher's microsecond.
inline Tensor make(at::IntArrayRef sizes, at::ScalarType type, const Tensor& x) { return at::detail::empty_cuda(sizes, type, x.device(), std::nullopt); }

inline uint8_t* bytes(const Tensor& t) { return static_cast<uint8_t*>(t.data_ptr()); }

}  // namespace

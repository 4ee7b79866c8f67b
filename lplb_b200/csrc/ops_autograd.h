// What the operators with gradients share: when a call is recorded, and what its gradients may be used for.
#pragma once

#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/variable.h>

#include <initializer_list>
#include <memory>
#include <unordered_set>
#include <vector>

#include "ops_check.h"

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Whether the call is recorded; arguments with a forward-mode tangent are refused.  Inside a capture a leaf whose gradient is
// collected on the default stream, because a graph that was recorded there still lives, is refused: the backward pass would make that
// stream wait for the captured one, which breaks the capture off with an error that names neither.
inline bool wants_grad(std::initializer_list<const Tensor*> tensors, const char* who) {
  for (const Tensor* t : tensors) check_no_tangent(*t, who);
  if (!at::GradMode::is_enabled()) return false;
  const Tensor* wanted = nullptr;
  for (const Tensor* t : tensors)
    if (wanted == nullptr && t->defined() && t->requires_grad()) wanted = t;
  if (wanted == nullptr) return false;
  {
    c10::cuda::OptionalCUDAGuard guard(at::device_of(*wanted));  // the stream that the call will run on, whatever device is current
    if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return true;
  }
  // leaves behind a weight's cast, a view or earlier operators too
  std::vector<std::shared_ptr<torch::autograd::Node>> held;  // leaves' own nodes, which nobody else may hold
  std::vector<torch::autograd::Node*> next;
  for (const Tensor* t : tensors) {
    if (!t->defined() || !t->requires_grad()) continue;
    if (!t->is_leaf()) {
      next.push_back(t->grad_fn().get());
    } else if (auto collects = torch::autograd::impl::try_get_grad_accumulator(*t)) {
      next.push_back(collects.get());
      held.push_back(std::move(collects));
    }
  }
  std::unordered_set<torch::autograd::Node*> seen;
  while (!next.empty()) {
    torch::autograd::Node* node = next.back();
    next.pop_back();
    if (!seen.insert(node).second) continue;
    if (dynamic_cast<torch::autograd::AccumulateGrad*>(node) != nullptr) {
      const auto stream = node->stream();
      if (stream && *stream == c10::cuda::getDefaultCUDAStream(stream->device_index()).unwrap())
        throw std::runtime_error(std::string("lplb_b200.ops.") + who +
                                 ": a graph recorded on the default stream still holds this leaf; delete its outputs before a backward pass is captured");
    }
    for (const auto& edge : node->next_edges())
      if (edge.function) next.push_back(edge.function.get());
  }
  return true;
}
inline Tensor or_none(const OptTensor& t) { return t ? *t : Tensor(); }
inline OptTensor or_none(const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; }

// Gradients as a backward pass returns them.  A pass that is itself recorded (create_graph=True) gets ones that refuse to be
// differentiated: these operators' gradients have none.
inline variable_list first_order(variable_list grads, const char* who) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list leaves;
  for (const Tensor& g : grads)
    if (g.defined()) leaves.push_back(g.detach().requires_grad_());
  if (leaves.empty()) return grads;
  auto refuse = std::make_shared<torch::autograd::DelayedError>(std::string("lplb_b200.ops.") + who + ": a gradient's gradient is not computed",
                                                                (int64_t)leaves.size());
  const variable_list marked = refuse->apply(std::move(leaves));
  size_t at = 0;
  for (Tensor& g : grads)
    if (g.defined()) g = marked[at++];
  return grads;
}

}  // namespace

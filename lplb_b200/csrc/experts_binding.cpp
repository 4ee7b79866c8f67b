// Python binding of the router's choice and of rows sorted by expert: checks of the arguments, outputs, launches on the current
// stream of the arguments' device.  The reference has no operators of this kind.
#include "experts_api.h"

#include "ops_autograd.h"

namespace {

using lplb::ops::CombineRows;
using lplb::ops::Gate;

// ---- the router's choice ----------------------------------------------------------------------------
Gate gate_args(const Tensor& logits, int64_t topk, bool sigmoid, bool renormalize, double scale) {
  OPS_CHECK(logits.is_cuda() && logits.dim() == 2, "gate_topk: logits must be a CUDA tensor [tokens, experts]");
  const int64_t tokens = logits.size(0), experts = logits.size(1);
  OPS_CHECK(experts >= 1 && experts <= lplb::ops::kGateMaxExperts, "gate_topk: 1 to " + text(lplb::ops::kGateMaxExperts) + " experts");
  OPS_CHECK(topk >= 1 && topk <= lplb::ops::kGateMaxTopk && topk <= experts,
            "gate_topk: topk must be 1 to " + text(lplb::ops::kGateMaxTopk) + ", and no more than there are experts");
  OPS_CHECK(tokens <= INT32_MAX, "gate_topk: fewer than 2^31 tokens");
  Gate g{};
  g.type = type_of(logits, "gate_topk: logits");
  g.logits = logits.data_ptr();
  g.ld = logits.stride(0);
  g.tokens = tokens;
  g.experts = (int)experts;
  g.topk = (int)topk;
  g.sigmoid = sigmoid;
  g.renormalize = renormalize;
  g.scale = (float)scale;
  return g;
}
Tensor rows_together(const Tensor& t) { return t.size(-1) < 2 || t.stride(-1) == 1 ? t : t.contiguous(); }

variable_list gate_forward(const Tensor& logits, int64_t topk, bool sigmoid, bool renormalize, double scale) {
  OPS_CHECK(logits.dim() == 2, "gate_topk: logits must be a CUDA tensor [tokens, experts]");
  c10::cuda::OptionalCUDAGuard guard(at::device_of(logits));
  const Tensor x = rows_together(logits);
  auto g = gate_args(x, topk, sigmoid, renormalize, scale);
  auto weights = make({g.tokens, topk}, torch::kFloat32, x), idx = make({g.tokens, topk}, torch::kInt64, x);
  g.weights = weights.data_ptr<float>();
  g.idx = idx.data_ptr<int64_t>();
  OPS_CUDA(lplb::ops::launch_gate(g, stream_of(x.get_device())));
  return {weights, idx};
}

Tensor gate_backward(const Tensor& logits, const Tensor& idx, const Tensor& dweights, bool sigmoid, bool renormalize, double scale) {
  c10::cuda::OptionalCUDAGuard guard(at::device_of(logits));
  const Tensor x = rows_together(logits), d = as_stored(dweights).contiguous();
  auto g = gate_args(x, idx.size(1), sigmoid, renormalize, scale);
  OPS_CHECK(idx.device() == x.device() && d.device() == x.device() && idx.scalar_type() == torch::kInt64 && idx.is_contiguous() &&
                idx.size(0) == g.tokens && d.scalar_type() == torch::kFloat32 && d.sizes() == idx.sizes(),
            "gate_topk: the weights' gradient must be float32, of the weights' shape, on the logits' device");
  auto dlogits = make(x.sizes(), x.scalar_type(), x);
  g.idx = idx.data_ptr<int64_t>();
  g.dweights = d.data_ptr<float>();
  g.dlogits = dlogits.data_ptr();
  OPS_CUDA(lplb::ops::launch_gate_backward(g, stream_of(x.get_device())));
  return dlogits;
}

struct GateTopk : torch::autograd::Function<GateTopk> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, int64_t topk, bool sigmoid, bool renormalize, double scale) {
    auto out = gate_forward(logits, topk, sigmoid, renormalize, scale);
    ctx->save_for_backward({logits, out[1]});
    ctx->mark_non_differentiable({out[1]});
    ctx->saved_data["sigmoid"] = sigmoid;
    ctx->saved_data["renormalize"] = renormalize;
    ctx->saved_data["scale"] = scale;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    Tensor dlogits;
    if (grads[0].defined())
      dlogits = gate_backward(saved[0], saved[1], grads[0], ctx->saved_data["sigmoid"].toBool(), ctx->saved_data["renormalize"].toBool(),
                              ctx->saved_data["scale"].toDouble());
    return first_order({dlogits, Tensor(), Tensor(), Tensor(), Tensor()}, "gate_topk");
  }
};

py::tuple gate_topk(const Tensor& given, int64_t topk, bool sigmoid, bool renormalize, double scale) {
  const Tensor logits = as_stored(given);
  const auto out = wants_grad({&logits}, "gate_topk") ? GateTopk::apply(logits, topk, sigmoid, renormalize, scale) : gate_forward(logits, topk, sigmoid, renormalize, scale);
  return py::make_tuple(out[0], out[1]);
}

// ---- rows sorted by expert ----------------------------------------------------------------------------
py::tuple expert_order(const Tensor& idx, int64_t experts) {
  OPS_CHECK(idx.is_cuda() && idx.dim() == 2 && (idx.scalar_type() == torch::kInt64 || idx.scalar_type() == torch::kInt32),
            "expert_order: idx must be a CUDA tensor [tokens, topk] of int64 or int32");
  OPS_CHECK(experts >= 1 && experts <= lplb::ops::kOrderMaxExperts, "expert_order: 1 to " + text(lplb::ops::kOrderMaxExperts) + " experts");
  OPS_CHECK(idx.size(1) >= 1 && idx.size(1) <= lplb::ops::kOrderMaxTopk, "expert_order: 1 to " + text(lplb::ops::kOrderMaxTopk) + " choices per token");
  OPS_CHECK(idx.numel() <= INT32_MAX, "expert_order: fewer than 2^31 choices in all");
  c10::cuda::CUDAGuard guard(idx.device());
  const Tensor ids = idx.contiguous();
  auto counts = make({experts}, torch::kInt32, ids), place = make(ids.sizes(), torch::kInt32, ids), source = make({ids.numel()}, torch::kInt32, ids);
  lplb::ops::Order o{};
  o.idx = ids.data_ptr();
  o.counts = counts.data_ptr<int>();
  o.place = place.data_ptr<int>();
  o.source = source.data_ptr<int>();
  o.pairs = ids.numel();
  o.experts = (int)experts;
  o.is64 = ids.scalar_type() == torch::kInt64;
  OPS_CUDA(lplb::ops::launch_order(o, ids.get_device(), stream_of(ids.get_device())));
  return py::make_tuple(counts, place, source);
}

void check_order(const Tensor& rows_or_tokens, const Tensor& place, const Tensor& source, const char* who) {
  OPS_CHECK(place.device() == rows_or_tokens.device() && place.dim() == 2 && place.scalar_type() == torch::kInt32 && place.is_contiguous() &&
                source.device() == rows_or_tokens.device() && source.dim() == 1 && source.scalar_type() == torch::kInt32 && source.is_contiguous() &&
                source.numel() == place.numel() && place.size(1) >= 1,
            who + std::string(": order must be one of expert_order's, on the same device"));
}

Tensor take_forward(const Tensor& x, const Tensor& place, const Tensor& source) {
  OPS_CHECK(x.is_cuda() && x.dim() == 2, "take_rows: x must be a CUDA tensor [tokens, values]");
  check_order(x, place, source, "take_rows");
  OPS_CHECK(place.size(0) == x.size(0), "take_rows: x must have a row for each of the order's tokens");
  OPS_CHECK(x.size(1) >= 1 && x.size(1) <= INT32_MAX / 16, "take_rows: rows without values, or too long");
  c10::cuda::CUDAGuard guard(x.device());
  const Tensor from = rows_together(x);
  auto rows = make({place.numel(), x.size(1)}, x.scalar_type(), x);
  lplb::ops::TakeRows t{};
  const int64_t size = x.element_size();
  t.x = from.data_ptr();
  t.place = place.data_ptr<int>();
  t.source = source.data_ptr<int>();
  t.rows = rows.data_ptr();
  t.ld_bytes = from.stride(0) * size;
  t.row_bytes = from.size(1) * size;
  t.tokens = from.size(0);
  t.topk = (int)place.size(1);
  OPS_CUDA(lplb::ops::launch_take_rows(t, sm_count(x.get_device()), stream_of(x.get_device())));
  return rows;
}

CombineRows combine_args(const Tensor& rows, const Tensor& place, const Tensor& source, const OptTensor& weights, const char* who) {
  OPS_CHECK(rows.is_cuda() && rows.dim() == 2, who + std::string(": rows must be a CUDA tensor [tokens * topk, values]"));
  check_order(rows, place, source, who);
  OPS_CHECK(rows.size(0) == place.numel(), who + std::string(": rows must have one for each of the order's choices"));
  OPS_CHECK(rows.size(1) >= 1 && rows.size(1) <= INT32_MAX / 16, who + std::string(": rows without values, or too long"));
  OPS_CHECK(!weights || (weights->device() == rows.device() && weights->scalar_type() == torch::kFloat32 && weights->sizes() == place.sizes() &&
                         weights->is_contiguous()),
            who + std::string(": weights must be [tokens, topk] on the rows' device"));
  CombineRows c{};
  c.type = type_of(rows, who);
  c.rows = rows.data_ptr();
  c.place = place.data_ptr<int>();
  c.source = source.data_ptr<int>();
  c.weights = weights ? weights->data_ptr<float>() : nullptr;
  c.ld = rows.stride(0);
  c.tokens = place.size(0);
  c.cols = (int)rows.size(1);
  c.topk = (int)place.size(1);
  return c;
}

Tensor combine_forward(const Tensor& rows, const Tensor& place, const Tensor& source, const OptTensor& weights) {
  OPS_CHECK(rows.dim() == 2, "combine_rows: rows must be a CUDA tensor [tokens * topk, values]");
  c10::cuda::OptionalCUDAGuard guard(at::device_of(rows));
  const Tensor from = rows_together(rows);
  auto c = combine_args(from, place, source, weights, "combine_rows");
  auto out = make({c.tokens, rows.size(1)}, rows.scalar_type(), rows);
  c.out = out.data_ptr();
  OPS_CUDA(lplb::ops::launch_combine_rows(c, sm_count(rows.get_device()), stream_of(rows.get_device())));
  return out;
}

variable_list combine_backward(const Tensor& dout, const Tensor& rows, const Tensor& place, const Tensor& source, const Tensor& weights,
                                bool need_rows, bool need_weights) {
  c10::cuda::OptionalCUDAGuard guard(at::device_of(rows));
  const Tensor from = rows_together(rows), d = rows_together(as_stored(dout));
  auto c = combine_args(from, place, source, weights, "combine_rows");
  OPS_CHECK(d.device() == rows.device() && d.dim() == 2 && d.size(0) == c.tokens && d.size(1) == c.cols && d.scalar_type() == rows.scalar_type(),
            "combine_rows: the gradient must be of the output's shape, type and device");
  Tensor drows, dweights;
  if (need_rows) {
    drows = make({rows.size(0), rows.size(1)}, rows.scalar_type(), rows);
    c.drows = drows.data_ptr();
  }
  if (need_weights) {
    dweights = make(place.sizes(), torch::kFloat32, rows);
    c.dweights = dweights.data_ptr<float>();
  }
  c.dout = d.data_ptr();
  c.dout_ld = d.stride(0);
  OPS_CUDA(lplb::ops::launch_combine_rows_backward(c, sm_count(rows.get_device()), stream_of(rows.get_device())));
  return {drows, dweights};
}

struct TakeRows : torch::autograd::Function<TakeRows> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& place, const Tensor& source) {
    ctx->save_for_backward({place, source});
    return take_forward(x, place, source);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    return first_order({combine_forward(as_stored(grads[0]), saved[0], saved[1], std::nullopt), Tensor(), Tensor()}, "take_rows");
  }
};

struct Combine : torch::autograd::Function<Combine> {
  static Tensor forward(AutogradContext* ctx, const Tensor& rows, const Tensor& place, const Tensor& source, const Tensor& weights) {
    ctx->save_for_backward({place, source, weights, rows});
    return combine_forward(rows, place, source, weights);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const auto found = combine_backward(grads[0], saved[3], saved[0], saved[1], saved[2], ctx->needs_input_grad(0), ctx->needs_input_grad(3));
    return first_order({found[0], Tensor(), Tensor(), found[1]}, "combine_rows");
  }
};
// without weights the gradient is take_rows, and no row is kept
struct Gather : torch::autograd::Function<Gather> {
  static Tensor forward(AutogradContext* ctx, const Tensor& rows, const Tensor& place, const Tensor& source) {
    ctx->save_for_backward({place, source});
    return combine_forward(rows, place, source, std::nullopt);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    return first_order({take_forward(as_stored(grads[0]), saved[0], saved[1]), Tensor(), Tensor()}, "combine_rows");
  }
};

Tensor take_rows(const Tensor& given, const Tensor& given_place, const Tensor& given_source) {
  const Tensor x = as_stored(given), place = in_a_row(given_place), source = in_a_row(given_source);
  if (!wants_grad({&x}, "take_rows")) return take_forward(x, place, source);
  type_of(x, "take_rows: x that requires a gradient");
  return TakeRows::apply(x, place, source);
}

Tensor combine_rows(const Tensor& given, const Tensor& given_place, const Tensor& given_source, const OptTensor& weights) {
  const Tensor rows = as_stored(given), place = in_a_row(given_place), source = in_a_row(given_source);
  if (!weights) return wants_grad({&rows}, "combine_rows") ? Gather::apply(rows, place, source) : combine_forward(rows, place, source, std::nullopt);
  OPS_CHECK(weights->is_floating_point(), "combine_rows: weights must be floating point [tokens, topk] on the rows' device");
  const Tensor w = as_stored(*weights).to(torch::kFloat32).contiguous();
  return wants_grad({&rows, &w}, "combine_rows") ? Combine::apply(rows, place, source, w) : combine_forward(rows, place, source, w);
}

}  // namespace

void bind_expert_ops(py::module_& m) {
  m.def("gate_topk", &gate_topk);
  m.def("expert_order", &expert_order);
  m.def("take_rows", &take_rows);
  m.def("combine_rows", &combine_rows);
  m.attr("GATE_MAX_EXPERTS") = lplb::ops::kGateMaxExperts;
  m.attr("GATE_MAX_TOPK") = lplb::ops::kGateMaxTopk;
  m.attr("ORDER_MAX_EXPERTS") = lplb::ops::kOrderMaxExperts;
}

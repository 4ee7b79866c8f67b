// Python binding of the product with an epilogue and of its gradients: checks of the arguments, outputs, launches on the current
// stream of the arguments' device.  The reference has no operators of this kind.
#include "matmul_api.h"

#include "ops_autograd.h"

namespace {

using lplb::ops::Activation;
using lplb::ops::Type;

int64_t up_to(int64_t n, int64_t step) { return (n + step - 1) / step * step; }
bool on_boundary(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }

// Rows that TMA can read: values of a row next to one another, every row on a 16-byte boundary; others are copied.
Tensor rows_for_tma(const Tensor& t) {
  const int64_t m = t.size(0), k = t.size(1);
  if ((t.stride(1) == 1 || k == 1) && on_boundary(t) && (m < 2 || (t.stride(0) * t.element_size() % 16 == 0 && t.stride(0) >= k))) return t;
  if (t.size(1) * t.element_size() % 16 == 0) {
    const Tensor c = t.contiguous();
    return on_boundary(c) ? c : c.clone();
  }
  auto wide = make({m, up_to(k, 16 / t.element_size())}, t.scalar_type(), t).narrow(1, 0, k);
  wide.copy_(t);
  return wide;
}
int64_t ld_of(const Tensor& t) { return t.size(0) < 2 ? up_to(t.size(1), 8) : t.stride(0); }
Tensor rows_together(const Tensor& t) { return t.size(-1) < 2 || t.stride(-1) == 1 ? t : t.contiguous(); }

struct Shape {
  int64_t m, n, k, groups;
};
Shape check_operands(const Tensor& a, const Tensor& b, const OptTensor& rows) {
  const auto device = a.device();
  const int64_t lead = rows ? 1 : 0;  // dimensions in front of a matrix
  OPS_CHECK(a.is_cuda() && a.dim() == 2 && (a.scalar_type() == torch::kBFloat16 || a.scalar_type() == torch::kFloat16),
            "matmul: a must be a CUDA tensor [rows, k] of bfloat16 or float16");
  OPS_CHECK(b.device() == device && b.dim() == 2 + lead && b.scalar_type() == a.scalar_type(),
            "matmul: b must be [n, k] (with rows: [groups, n, k]) of a's type on a's device");
  Shape s{a.size(0), b.size(-2), a.size(1), rows ? b.size(0) : 1};
  OPS_CHECK(s.groups >= 1 && s.groups <= lplb::ops::kMatmulMaxGroups, "matmul: 1 to " + text(lplb::ops::kMatmulMaxGroups) + " groups");
  OPS_CHECK(!rows || (rows->device() == device && rows->scalar_type() == torch::kInt32 && rows->dim() == 1 && rows->size(0) == s.groups && rows->is_contiguous()),
            "matmul: rows must be contiguous int32, one number for each matrix of b, on a's device");
  OPS_CHECK(s.m <= lplb::ops::kMaxRows && s.groups * s.n <= lplb::ops::kMaxRows,
            "matmul: at most " + text(lplb::ops::kMaxRows) + " rows of a, and of all matrices of b together");
  OPS_CHECK(s.k >= 8 && s.k % 8 == 0 && s.k <= (1 << 28) && b.size(-1) == s.k, "matmul: a and b must have the same k, a multiple of 8");
  OPS_CHECK(s.n >= 1 && s.n <= (1 << 28), "matmul: b has no rows, or too many");
  OPS_CHECK(b.is_contiguous() && on_boundary(b), "matmul: b must be contiguous and start on a 16-byte boundary");
  return s;
}
Activation activation_of(int64_t code, const Shape& s) {
  const auto act = static_cast<Activation>(code);
  OPS_CHECK(act != lplb::ops::kSwiglu || s.n % (2 * lplb::ops::kGateBlock) == 0,
            "matmul: 'swiglu' needs blocks of 128 gate rows and their 128 up rows: n must be a multiple of 256");
  return act;
}
const int* rows_of(const OptTensor& rows) { return rows ? rows->data_ptr<int>() : nullptr; }

// (out, pre): pre is the sum before the activation, in 32 bits, where `keep`
variable_list run_forward(const Tensor& a, const Tensor& b, const OptTensor& bias, int64_t activation, const OptTensor& residual, const OptTensor& rows,
                      bool out_f32, bool keep) {
  const Shape s = check_operands(a, b, rows);
  lplb::ops::Matmul p{};
  p.activation = activation_of(activation, s);
  const int64_t cols = p.activation == lplb::ops::kSwiglu ? s.n / 2 : s.n;
  const auto type = out_f32 ? torch::kFloat32 : a.scalar_type();
  OPS_CHECK(!bias || (bias->device() == a.device() && (bias->scalar_type() == a.scalar_type() || bias->scalar_type() == torch::kFloat32) &&
                      bias->dim() == b.dim() - 1 && bias->size(-1) == s.n && bias->numel() == s.groups * s.n),
            "matmul: bias must be [n] (with rows: [groups, n]) of a's type or float32 on a's device");
  OPS_CHECK(!residual || (residual->device() == a.device() && residual->scalar_type() == type && residual->dim() == 2 && residual->size(0) == s.m &&
                          residual->size(1) == cols),
            "matmul: residual must be of the output's shape, type and device");
  c10::cuda::CUDAGuard guard(a.device());
  const Tensor from = rows_for_tma(a);
  const Tensor added = bias ? bias->contiguous() : Tensor(), carried = residual ? rows_together(*residual) : Tensor();
  auto out = make({s.m, cols}, type, a);
  Tensor pre;
  p.a = from.data_ptr();
  p.b = b.data_ptr();
  p.rows = rows_of(rows);
  p.out = out.data_ptr();
  p.m = s.m;
  p.n = s.n;
  p.k = s.k;
  p.a_ld = ld_of(from);
  p.out_ld = cols;
  p.groups = (int)s.groups;
  p.type = type_of(a, "matmul: a");
  p.out_type = out_f32 ? Type::kF32 : p.type;
  if (bias) {
    p.bias = added.data_ptr();
    p.bias_type = type_of(added, "matmul: bias");
  }
  if (residual) {
    p.residual = carried.data_ptr();
    p.residual_ld = carried.stride(0);
  }
  if (keep) {
    pre = make({s.m, up_to(s.n, 4)}, torch::kFloat32, a);
    p.pre = pre.data_ptr<float>();
    p.pre_ld = pre.size(1);
  }
  OPS_CUDA(lplb::ops::launch_matmul(p, a.get_device(), stream_of(a.get_device())));
  return {out, pre};
}

// (da, db, dbias), each where it is needed.  bias: its type, float32 or a's.
variable_list run_backward(const Tensor& given, const Tensor& a, const Tensor& b, const OptTensor& pre, int64_t activation, const OptTensor& rows, bool out_f32,
                       bool bias_f32, bool need_a, bool need_b, bool need_bias) {
  const Shape s = check_operands(a, b, rows);
  const auto act = activation_of(activation, s);
  const Tensor dout = as_stored(given);
  const int64_t cols = act == lplb::ops::kSwiglu ? s.n / 2 : s.n;
  const auto out_type = out_f32 ? torch::kFloat32 : a.scalar_type();
  OPS_CHECK(dout.device() == a.device() && dout.scalar_type() == out_type && dout.dim() == 2 && dout.size(0) == s.m && dout.size(1) == cols,
            "matmul: the gradient must be of the output's shape, type and device");
  OPS_CHECK((act == lplb::ops::kNoActivation) == !pre, "matmul: an activation's gradient needs what it was taken of");
  c10::cuda::CUDAGuard guard(a.device());
  const int device = a.get_device();
  const auto stream = stream_of(device);
  const auto type = type_of(a, "matmul: a");
  Tensor da, db, dbias;
  if (need_a) da = make({s.m, s.k}, a.scalar_type(), a);
  if (need_b) db = make(b.sizes(), b.scalar_type(), a);
  if (need_bias) {
    auto shape = b.sizes().vec();
    shape.pop_back();
    dbias = make(shape, bias_f32 ? torch::kFloat32 : a.scalar_type(), a);
  }
  if (s.m == 0) {
    if (need_b) db.zero_();
    if (need_bias) dbias.zero_();
  } else {
    // without an activation dz is dout, where the products can read it
    const bool same = act == lplb::ops::kNoActivation && !out_f32;
    Tensor dz = same ? rows_for_tma(dout) : Tensor(), dz_weight = dz;
    Tensor row_most, column_most;  // of dz in float16, which is stored in parts of a power of two
    if (!same || need_bias) {
      const Tensor d = rows_together(dout);
      lplb::ops::MatmulPre p{};
      if (!same && (need_a || need_b)) {
        const bool in_parts = type == Type::kF16;
        if (need_a || !in_parts) {
          dz = make({s.m, up_to(s.n, 8)}, a.scalar_type(), a);
          p.dz = dz.data_ptr();
        }
        dz_weight = dz;
        p.dz_ld = up_to(s.n, 8);
        if (in_parts && need_a) {
          row_most = make({s.m}, torch::kInt32, a);
          p.row_most = reinterpret_cast<uint32_t*>(row_most.data_ptr<int>());
        }
        if (in_parts && need_b) {
          dz_weight = make({s.m, up_to(s.n, 8)}, a.scalar_type(), a);
          p.dz_weight = dz_weight.data_ptr();
          column_most = make({s.groups, s.n}, torch::kInt32, a);
          p.column_most = reinterpret_cast<uint32_t*>(column_most.data_ptr<int>());
        }
      }
      p.dout = d.data_ptr();
      p.dout_ld = d.stride(0);
      if (pre) {
        p.pre = pre->data_ptr<float>();
        p.pre_ld = pre->size(1);
      }
      p.rows = rows_of(rows);
      p.m = s.m;
      p.n = s.n;
      p.groups = (int)s.groups;
      p.activation = act;
      p.type = type;
      p.out_type = out_f32 ? Type::kF32 : type;
      p.bias_type = bias_f32 ? Type::kF32 : type;
      Tensor parts;
      if (need_bias) {
        p.dbias = dbias.data_ptr();
        int64_t floats = 0;
        int splits = 0;
        OPS_CUDA(lplb::ops::matmul_pre_parts(p, device, &floats, &splits));
        if (floats > 0) {
          parts = make({floats}, torch::kFloat32, a);
          p.parts = parts.data_ptr<float>();
        }
      }
      OPS_CUDA(lplb::ops::launch_matmul_pre(p, device, stream));
    }
    if (need_a) {
      lplb::ops::MatmulInput p{};
      p.dz = dz.data_ptr();
      p.most = row_most.defined() ? reinterpret_cast<const uint32_t*>(row_most.data_ptr<int>()) : nullptr;
      p.b = b.data_ptr();
      p.rows = rows_of(rows);
      p.da = da.data_ptr();
      p.m = s.m;
      p.n = s.n;
      p.k = s.k;
      p.dz_ld = ld_of(dz);
      p.da_ld = s.k;
      p.groups = (int)s.groups;
      p.type = type;
      OPS_CUDA(lplb::ops::launch_matmul_input(p, device, stream));
    }
    if (need_b) {
      const Tensor from = rows_for_tma(a);
      lplb::ops::MatmulWeight p{};
      p.dz = dz_weight.data_ptr();
      p.most = column_most.defined() ? reinterpret_cast<const uint32_t*>(column_most.data_ptr<int>()) : nullptr;
      p.a = from.data_ptr();
      p.rows = rows_of(rows);
      p.db = db.data_ptr();
      p.m = s.m;
      p.n = s.n;
      p.k = s.k;
      p.dz_ld = ld_of(dz_weight);
      p.a_ld = ld_of(from);
      p.groups = (int)s.groups;
      p.type = type;
      Tensor copies;  // of this call alone: calls on two streams, or two captured graphs, share nothing
      if (rows) {
        copies = make({lplb::ops::matmul_weight_copies(p)}, torch::kUInt8, a);
        p.copies = copies.data_ptr();
      }
      OPS_CUDA(lplb::ops::launch_matmul_weight(p, device, stream));
    }
  }
  return {da, db, dbias};
}

struct Product : torch::autograd::Function<Product> {
  static Tensor forward(AutogradContext* ctx, const Tensor& a, const Tensor& b, const OptTensor& bias, const OptTensor& residual, const OptTensor& rows,
                        int64_t activation, bool out_f32) {
    const bool keep = activation != lplb::ops::kNoActivation && (a.requires_grad() || b.requires_grad() || (bias && bias->requires_grad()));
    const auto out = run_forward(a, b, bias, activation, residual, rows, out_f32, keep);
    ctx->save_for_backward({a, b, or_none(rows), out[1]});
    ctx->saved_data["activation"] = activation;
    ctx->saved_data["out_f32"] = out_f32;
    ctx->saved_data["bias"] = bias.has_value();
    ctx->saved_data["bias_f32"] = bias && bias->scalar_type() == torch::kFloat32;
    ctx->saved_data["residual"] = residual.has_value();
    return out[0];
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const bool has_bias = ctx->saved_data["bias"].toBool();
    // the tensors that there are, in their order
    const bool need_a = ctx->needs_input_grad(0), need_b = ctx->needs_input_grad(1), need_bias = has_bias && ctx->needs_input_grad(2);
    const bool need_residual = ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(has_bias ? 3 : 2);
    variable_list found(3);
    if (need_a || need_b || need_bias)
      found = run_backward(grads[0], saved[0], saved[1], or_none(saved[3]), ctx->saved_data["activation"].toInt(), or_none(saved[2]),
                         ctx->saved_data["out_f32"].toBool(), ctx->saved_data["bias_f32"].toBool(), need_a, need_b, need_bias);
    return first_order({found[0], found[1], found[2], need_residual ? grads[0] : Tensor(), Tensor(), Tensor(), Tensor()}, "matmul");
  }
};

Tensor matmul(const Tensor& given_a, const Tensor& given_b, const OptTensor& given_bias, int64_t activation, const OptTensor& given_residual,
              const OptTensor& given_rows, bool out_f32) {
  const Tensor a = as_stored(given_a), b = as_stored(given_b);
  const OptTensor rows = given_rows ? OptTensor(in_a_row(*given_rows)) : std::nullopt;
  const OptTensor bias = as_stored(given_bias), residual = as_stored(given_residual);
  const Tensor added = or_none(bias), carried = or_none(residual);
  if (wants_grad({&a, &b, &added, &carried}, "matmul")) return Product::apply(a, b, bias, residual, rows, activation, out_f32);
  return run_forward(a, b, bias, activation, residual, rows, out_f32, false)[0];
}

}  // namespace

void bind_matmul(py::module_& m) {
  m.def("matmul", &matmul);
  m.attr("MATMUL_MAX_GROUPS") = lplb::ops::kMatmulMaxGroups;
}

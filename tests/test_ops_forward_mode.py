"""Forward-mode differentiation: the operators' plain statements carry a tangent, the kernels have none and refuse it."""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from lplb_b200 import ops

F32, BF16 = torch.float32, torch.bfloat16


def _calls(device):
    """name -> (function of one tensor, the tensor)"""
    g = torch.Generator().manual_seed(0)
    normal = lambda *shape: torch.randn(*shape, generator=g).to(device)  # noqa: E731
    order = ops.expert_order(torch.tensor([[0, 1], [1, -1], [2, 0]], device=device), 3)
    x, rows, w, b = normal(3, 8), normal(6, 8), normal(3, 2), normal(16, 8).bfloat16()
    a, bias, residual = normal(3, 8).bfloat16(), normal(16), normal(3, 16)
    product = dict(a=a, b=b, bias=bias, activation="silu", residual=residual, out_dtype=F32)
    return {
        "gate_topk": (lambda t: ops.gate_topk(t, 2, "sigmoid")[0], x),
        "take_rows": (lambda t: ops.take_rows(t, order), x),
        "combine_rows: rows": (lambda t: ops.combine_rows(t, order, w), rows),
        "combine_rows: weights": (lambda t: ops.combine_rows(rows, order, t), w),
        "combine_rows: weights in 64 bits": (lambda t: ops.combine_rows(rows, order, t), w.double()),
        "combine_rows without weights": (lambda t: ops.combine_rows(t, order), rows),
        **{f"matmul: {name}": (lambda t, name=name: ops.matmul(**{**product, name: t}), product[name]) for name in ("a", "b", "bias", "residual")},
    }


NAMES = list(_calls("cpu"))


@pytest.mark.parametrize("name", NAMES)
def test_the_plain_statements_carry_a_tangent(name):
    f, x = _calls("cpu")[name]
    t = torch.randn(x.shape, generator=torch.Generator().manual_seed(1)).to(x.dtype)
    with forward_ad.dual_level():
        got = forward_ad.unpack_dual(f(forward_ad.make_dual(x, t))).tangent
    assert got is not None and got.any()
    # against the gradient's: <f'(x) t, v> = <t, f'(x)^T v>; everything is rounded to bfloat16 at most a few times
    leaf = x.clone().requires_grad_()
    v = torch.randn(got.shape, generator=torch.Generator().manual_seed(2))
    (dx,) = torch.autograd.grad(f(leaf), leaf, v.to(got.dtype))
    one, other = (got.double() * v.double()).sum(), (t.double() * dx.double()).sum()
    size = (got.double() * v.double()).abs().sum() + (t.double() * dx.double()).abs().sum()
    assert abs(one - other) <= 2.0**-7 * size


@pytest.mark.gpu
@pytest.mark.parametrize("grad_mode", [True, False])
@pytest.mark.parametrize("name", NAMES)
def test_the_kernels_refuse_a_tangent(name, grad_mode):
    f, x = _calls("cuda")[name]
    with torch.set_grad_enabled(grad_mode):
        plain = f(x)
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(x, torch.ones_like(x))
            with pytest.raises(ValueError, match="forward-mode tangent"):
                f(dual)
            assert torch.equal(f(forward_ad.unpack_dual(dual).primal), plain)  # without it
        with pytest.raises((ValueError, RuntimeError)):
            torch.func.jvp(f, (x,), (torch.ones_like(x),))
        assert torch.equal(f(x), plain)


@pytest.mark.gpu
def test_the_8_bit_operators_refuse_a_tangent():
    x, w = torch.randn(4, 256, device="cuda"), torch.randn(256, device="cuda")
    calls = [
        lambda t: ops.quantize_fp8(t),
        lambda t: ops.quantize_weight_fp8(t),
        lambda t: ops.rms_norm_fp8(t, w),
        lambda t: ops.rms_norm_fp8(x, w, t),
    ]
    with forward_ad.dual_level():
        for call in calls:
            call(x)
            with pytest.raises(ValueError, match="forward-mode tangent"):
                call(forward_ad.make_dual(x, torch.ones_like(x)))
        with pytest.raises(ValueError, match="forward-mode tangent"):
            ops.rms_norm_fp8(x, forward_ad.make_dual(w, torch.ones_like(w)))

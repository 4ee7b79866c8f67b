"""Lazily conjugated and negated views, whose memory holds other values than they stand for: operators read the values."""

import pytest
import torch

from lplb_b200 import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
F32, F16 = torch.float32, torch.float16


def _negated(*shape, dtype, device, seed=0):
    """A lazily negated view of float16 or float32: the imaginary part of a conjugate."""
    g = torch.Generator().manual_seed(seed)
    t = torch.randn(*shape, 2, generator=g).to(dtype)
    view = torch.view_as_complex(t.to(device)).conj().imag
    assert view.is_neg()
    return view


def _order(device):
    return ops.expert_order(torch.tensor([[0, 1], [1, -1], [2, 0]], device=device), 3)


def _calls(device):
    """name -> (function of lazily negated tensors, those)"""
    neg = lambda *shape, dtype=F32, seed=0: _negated(*shape, dtype=dtype, device=device, seed=seed)  # noqa: E731
    order = _order(device)
    a, b = neg(3, 16, dtype=F16, seed=1), neg(8, 16, dtype=F16, seed=2).mul(1)  # (b has to be contiguous)
    plain = lambda t: t.clone().resolve_neg()  # noqa: E731
    lazily = lambda t: torch._neg_view(-t)  # noqa: E731  contiguous, and lazily negated
    return {
        "gate_topk": (lambda x: ops.gate_topk(x, 2, "sigmoid")[0], (neg(3, 8),)),
        "take_rows": (lambda x: ops.take_rows(x, order), (neg(3, 8),)),
        "combine_rows": (lambda y, w: ops.combine_rows(y, order, w), (neg(6, 8), neg(3, 2, seed=1))),
        "combine_rows without weights": (lambda y: ops.combine_rows(y, order), (neg(6, 8),)),
        "matmul": (lambda a, b, bias, r: ops.matmul(a, b, bias, "silu", r, out_dtype=F32), (a, lazily(plain(b)), neg(8, seed=3), neg(3, 8, seed=4))),
        "grouped matmul": (
            lambda a, b, bias: ops.matmul(a, b, bias, rows=torch.tensor([2, 1], dtype=torch.int32, device=device)),
            (a, lazily(torch.stack([plain(b), -plain(b)])), neg(2, 8, dtype=F16, seed=3)),
        ),
    }


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("name", list(_calls("cpu")))
def test_negated_arguments(name, device):
    f, args = _calls(device)[name]
    assert all(t.is_neg() for t in args)
    values = tuple(t.clone().resolve_neg().contiguous() for t in args)
    assert not any(t.is_neg() for t in values)
    assert torch.equal(f(*args), f(*values))
    # and through them to what they are views of
    lazy, plain = (tuple(t.detach().clone().requires_grad_() for t in values) for _ in range(2))
    out, want = f(*(torch._neg_view(t) for t in lazy)), f(*(-t for t in plain))
    v = torch.randn(out.shape, generator=torch.Generator().manual_seed(9)).to(out.dtype).to(device)
    assert torch.equal(out, want)
    for got, right in zip(torch.autograd.grad(out, lazy, v), torch.autograd.grad(want, plain, v)):
        assert torch.equal(got, right)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("name", list(_calls("cpu")))
def test_a_gradient_that_arrives_negated(name, device):
    f, args = _calls(device)[name]
    leaves = tuple(t.clone().resolve_neg().contiguous().requires_grad_() for t in args)
    out = f(*leaves)
    d = torch.randn(out.shape, generator=torch.Generator().manual_seed(9)).to(out.dtype).to(device)
    want = torch.autograd.grad(out, leaves, d, retain_graph=True)
    for got, right in zip(torch.autograd.grad(out, leaves, torch._neg_view(-d)), want):
        assert torch.equal(got, right)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.complex64, torch.complex128])
def test_rows_of_complex_numbers(dtype, device):
    z = torch.randn(3, 5, dtype=dtype, generator=torch.Generator().manual_seed(0)).to(device)
    order = _order(device)
    want = ops.take_rows(z.conj().resolve_conj(), order)
    assert torch.equal(ops.take_rows(z.conj(), order).resolve_conj(), want) and want.imag.any()
    assert torch.equal(ops.take_rows(z, order), want.conj().resolve_conj())


@pytest.mark.parametrize("device", DEVICES)
def test_8_bit_operators(device):
    x, w = _negated(4, 256, dtype=F32, device=device), _negated(256, dtype=F32, device=device, seed=1)
    rows = torch._neg_view(-x.clone().resolve_neg())  # values of a row next to one another, as these operators ask for
    weight = torch._neg_view(-w.clone().resolve_neg())
    assert rows.is_neg() and weight.is_neg()
    x, w = rows.clone().resolve_neg(), weight.clone().resolve_neg()
    as_bytes = lambda out: [t.view(torch.uint8) if t.element_size() == 1 else t for t in out]  # noqa: E731
    for got, want in (
        (ops.quantize_fp8(rows), ops.quantize_fp8(x)),
        (ops.quantize_weight_fp8(rows), ops.quantize_weight_fp8(x)),
        (ops.rms_norm_fp8(rows, weight, rows), ops.rms_norm_fp8(x, w, x)),
    ):
        for one, other in zip(as_bytes(got), as_bytes(want)):
            assert torch.equal(one, other)


@pytest.mark.gpu
def test_an_output_that_is_negated_is_refused():
    q, scale = ops.quantize_fp8(torch.randn(4, 256, device="cuda"))
    wq, w_scale = ops.quantize_weight_fp8(torch.randn(8, 256, device="cuda"))
    with pytest.raises(ValueError, match="negated"):
        ops.matmul_fp8(q, scale, wq, w_scale, out_dtype=F32, out=torch._neg_view(torch.zeros(4, 8, device="cuda")))


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [8, 100])
def test_weights_of_the_layer(tokens):
    from test_gpu_moe_inputs import _avail, _inputs, _layer

    layer = _layer(torch.bfloat16)
    x, idx, w = _inputs(tokens)
    view = torch._neg_view(-w)
    assert view.is_neg() and torch.equal(layer.forward(x, idx, view, _avail()), layer.forward(x, idx, w, _avail()))

"""The product with an epilogue on the CPU: the plain statements against the definition in 64 bits and against differences, and
refusals."""

import experts_oracle as oracle
import pytest
import torch

from lplb_b200 import ops

ACTIVATIONS = [None, "relu", "gelu", "silu", "swiglu"]


def make_case(m, n, k, groups, activation, bias, residual, dtype, out_dtype, seed, device="cpu"):
    """(arguments of matmul, dout); groups: None, or the rows of every matrix."""
    g = torch.Generator().manual_seed(seed)
    lead = () if groups is None else (len(groups),)
    cols = n // 2 if activation == "swiglu" else n
    args = {
        "a": torch.randn(m, k, generator=g).to(dtype),
        "b": (torch.randn(*lead, n, k, generator=g) * k**-0.5).to(dtype),
        "bias": torch.randn(*lead, n, generator=g).to(bias) if bias else None,
        "residual": torch.randn(m, cols, generator=g).to(out_dtype) if residual else None,
        "rows": None if groups is None else torch.tensor(groups, dtype=torch.int32),
    }
    args = {name: None if t is None else t.to(device) for name, t in args.items()}
    return {**args, "activation": activation, "out_dtype": out_dtype}, torch.randn(m, cols, generator=g).to(out_dtype).to(device)


def run(args, dout):
    """Everything that matmul gives: out and the gradients."""
    leaves = {name: t.clone().requires_grad_() for name, t in args.items() if name in ("a", "b", "bias", "residual") and t is not None}
    out = ops.matmul(**{**args, **leaves})
    grads = torch.autograd.grad(out, tuple(leaves.values()), dout)
    return {"out": out.detach(), **{"d" + name: g for name, g in zip(leaves, grads)}}


def compare(got, args, dout):
    want = oracle.product(
        args["a"], args["b"], args["bias"], args["activation"], args["residual"], args["rows"], dout, args["a"].dtype, args["out_dtype"]
    )
    assert set(got) == set(want)
    for name, (value, bound) in want.items():
        off = (got[name].double() - value).abs()
        assert (off <= bound).all(), (name, float((off / bound).max()))
    for name in ("a", "b", "bias", "residual"):
        assert args[name] is None or got["d" + name].dtype == args[name].dtype
    assert got["out"].dtype == args["out_dtype"]


@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("groups", [None, [3, 0, 5, -1, 2]])
@pytest.mark.parametrize("dtype,out_dtype,bias", [(torch.bfloat16, torch.bfloat16, torch.float32), (torch.float16, torch.float32, torch.float16)])
def test_product(activation, groups, dtype, out_dtype, bias):
    args, dout = make_case(13, 256, 40, groups, activation, bias, True, dtype, out_dtype, 3)
    compare(run(args, dout), args, dout)


def test_more_rows_than_there_are():
    args, dout = make_case(4, 6, 8, [3, 2**31 - 1, 7], "relu", torch.float32, False, torch.bfloat16, torch.bfloat16, 1)
    compare(run(args, dout), args, dout)


@pytest.mark.parametrize("activation", [a for a in ACTIVATIONS if a != "relu"])
def test_gradients_against_differences(activation):
    g = torch.Generator().manual_seed(0)
    n = 256 if activation == "swiglu" else 6
    rows = torch.tensor([2, 3], dtype=torch.int32)
    a, b, bias = torch.randn(6, 8, generator=g).double(), torch.randn(2, n, 8, generator=g).double(), torch.randn(2, n, generator=g).double()
    out, z = ops.reference.matmul_reference(a, b, bias, activation, None, rows)
    dout = torch.randn(out.shape, generator=g).double()
    grads = dict(zip(("a", "b", "bias"), ops.reference.matmul_backward_reference(dout, a, b, z, activation, rows)))
    given = {"a": a, "b": b, "bias": bias}

    def value(**changed):
        t = {**given, **changed}
        return (ops.reference.matmul_reference(t["a"], t["b"], t["bias"], activation, None, rows)[0] * dout).sum().item()

    h = 1e-5
    for name, at in [("a", (0, 0)), ("a", (4, 7)), ("a", (5, 1)), ("b", (0, 1, 3)), ("b", (1, 5, 0)), ("bias", (0, 2)), ("bias", (1, 4))]:
        step = torch.zeros_like(given[name])
        step[at] = h
        slope = (value(**{name: given[name] + step}) - value(**{name: given[name] - step})) / (2 * h)
        assert abs(slope - grads[name][at].item()) < 1e-6 * (1 + abs(slope)), (name, at)


def test_only_what_is_asked_for():
    args, dout = make_case(5, 12, 16, None, "gelu", torch.float32, True, torch.bfloat16, torch.bfloat16, 1)
    for name in ("a", "b", "bias", "residual"):
        leaf = args[name].clone().requires_grad_()
        ops.matmul(**{**args, name: leaf}).backward(dout)
        assert leaf.grad.shape == leaf.shape
    assert not ops.matmul(**args).requires_grad


def refusals(device):
    """(changed arguments, words of the refusal)"""
    def t(*shape, dtype=torch.bfloat16):
        return torch.zeros(*shape, dtype=dtype, device=device)

    rows = torch.tensor([1, 2], dtype=torch.int32, device=device)
    return [
        ({"activation": "tanh"}, "activation"),
        ({"out_dtype": torch.float16}, "out_dtype"),
        ({"a": t(4)}, "a must be"),
        ({"a": t(4, 16, dtype=torch.float32), "out_dtype": torch.float32}, "a must be"),
        ({"b": t(8, 16, dtype=torch.float16)}, "b must be"),
        ({"b": t(8, 24)}, "same k"),
        ({"a": t(4, 12), "b": t(8, 12)}, "multiple of 8"),
        ({"a": t(4, 0), "b": t(8, 0)}, "multiple of 8"),
        ({"b": t(16, 8).T}, "contiguous"),
        ({"b": t(0, 16)}, "no rows"),
        ({"activation": "swiglu"}, "256"),
        ({"bias": t(7)}, "bias"),
        ({"bias": t(1, 8)}, "bias"),
        ({"bias": t(8, dtype=torch.float16)}, "bias"),
        ({"residual": t(4, 7)}, "residual"),
        ({"residual": t(4, 8, dtype=torch.float32)}, "residual"),
        ({"rows": rows}, "b must be"),
        ({"rows": rows, "b": t(3, 8, 16)}, "rows"),
        ({"rows": rows.long(), "b": t(2, 8, 16)}, "rows"),
        ({"rows": rows[:0], "b": t(0, 8, 16)}, "groups"),
        ({"rows": torch.zeros(1025, dtype=torch.int32, device=device), "b": t(1025, 1, 16)}, "groups"),
        ({"rows": rows, "b": t(2, 8, 16), "bias": t(8)}, "bias"),
    ]


@pytest.mark.parametrize("number", range(22))
def test_refuses(number):
    changed, words = refusals("cpu")[number]
    good = {"a": torch.zeros(4, 16, dtype=torch.bfloat16), "b": torch.zeros(8, 16, dtype=torch.bfloat16)}
    assert ops.matmul(**good).shape == (4, 8)
    with pytest.raises(ValueError, match=words):
        ops.matmul(**{**good, **changed})


def test_all_refusals_are_tried():
    assert len(refusals("cpu")) == 22

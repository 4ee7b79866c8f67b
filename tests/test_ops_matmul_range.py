"""Gradients of the product in float16 whose way leads over values that float16 does not hold: finite gradients stay finite, and none is lost.

Bounds: a value of dz is rounded to half a step of float16 of itself, 2^-11, and where it is far below the largest of its row (or
column) by 2^-39 of that one; sums of n products are off by (n / 16 + 32) * 2^-23 of the sum of magnitudes; results are rounded once, to
2^-11 of themselves or 2^-25."""

import pytest
import torch
from experts_oracle import act, parts_of

from lplb_b200 import ops

F16, F32 = torch.float16, torch.float32
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
E = 2.0**-11


def _sums(terms):
    return (terms / 16 + 32) * 2.0**-23


def _make(kind, m, n, k, groups, seed):
    """(arguments of matmul, dout)"""
    g = torch.Generator().manual_seed(seed)
    lead = () if groups is None else (len(groups),)
    normal = lambda *shape: torch.randn(*shape, generator=g)  # noqa: E731
    a, b, cols = normal(m, k), normal(*lead, n, k), n // 2 if kind == "swiglu" else n
    dout = normal(m, cols)
    args = {"activation": None, "out_dtype": F32, "bias": None}
    if kind == "large":
        a, b, dout = 1e-3 * a, 1e-3 * b, 1e5 * dout
    elif kind == "small":
        a, b, dout = 100 * a, 100 * b, 2e-8 * dout
    elif kind == "rows":  # of 2^-30 to 1
        b, dout = 2.0**10 * b, dout * torch.exp2(torch.linspace(-30, 0, m)).unsqueeze(1)
    elif kind == "columns":
        a, dout = 2.0**10 * a, dout * torch.exp2(torch.linspace(-30, 0, n))
    elif kind == "swiglu":  # a large up value; everything that is given and returned is in float16
        a, b, dout = 5e-4 * a, 2e-4 * b, 1e4 * dout
        bias = torch.where(torch.arange(n) % 256 < 128, 0.0, 300.0)
        args = {"activation": "swiglu", "out_dtype": F16, "bias": bias.expand(*lead, n).contiguous()}
        dout = dout.half()
    args |= {"a": a.half(), "b": b.half(), "rows": None if groups is None else torch.tensor(groups, dtype=torch.int32)}
    return args, dout


def _gradients(args, dout, names=("a", "b")):
    leaves = {name: args[name].clone().requires_grad_() for name in names}
    return dict(zip(names, torch.autograd.grad(ops.matmul(**{**args, **leaves}), tuple(leaves.values()), dout)))


def _wanted(args, dout):
    """Values in 64 bits, and bounds."""
    a, b, rows, activation = args["a"].double(), args["b"].double(), args["rows"], args["activation"]
    (m, k), n = a.shape, b.shape[-2]
    z, z_err = a.new_zeros(m, n), a.new_zeros(m, n)
    for e, part in parts_of(m, rows):
        at = slice(None) if e is None else e
        z[part], z_err[part] = a[part] @ b[at].T, _sums(k) * (a[part].abs() @ b[at].abs().T)
        if args["bias"] is not None:
            z[part] += args["bias"][at].double()
    z_err += 2.0**-23 * z.abs()
    z.requires_grad_()
    (dz,) = torch.autograd.grad(act(z, activation), z, dout.double())
    dz_err = torch.zeros_like(dz)
    if activation == "swiglu":  # the slope's own error, as of a z that is kept in 32 bits
        (gate, up), (s_gate, s_up) = (t.detach().view(m, -1, 2, 128).unbind(2) for t in (z, z_err))
        d = dout.double().view(m, -1, 128).abs()
        to_gate = d * ((up.abs() + s_up) * s_gate + 1.13 * s_up + 2.0**-16 * (up.abs() + 1) * (gate.abs() + 1))
        dz_err = torch.stack((to_gate, d * (1.13 * s_gate + 2.0**-16 * gate.abs())), 2).reshape(m, -1)
    values = {"a": torch.zeros_like(a), "b": torch.zeros_like(b)}
    bounds = {name: torch.zeros_like(t) for name, t in values.items()}
    for e, part in parts_of(m, rows):
        if part.stop == part.start:
            continue
        at, d, err = slice(None) if e is None else e, dz[part], dz_err[part] + E * dz[part].abs()
        by_row, by_column = (err + 2.0**-39 * d.abs().amax(dim, keepdim=True) for dim in (1, 0))
        values["a"][part], values["b"][at] = d @ b[at], d.T @ a[part]
        bounds["a"][part] = by_row @ b[at].abs() + _sums(n) * (d.abs() @ b[at].abs())
        bounds["b"][at] = by_column.T @ a[part].abs() + _sums(part.stop - part.start) * (d.abs().T @ a[part].abs())
    return {name: (v, bounds[name] * (1 + E) + E * v.abs() + 2.0**-25) for name, v in values.items()}


CASES = [("large", 3, 5, 8, None), ("small", 3, 5, 8, None)] + [
    (kind, m, n, k, groups)
    for kind in ("large", "small", "rows", "columns", "swiglu")
    for m, n, k, groups in ((40, 256, 64, None), (300, 512, 136, [100, 0, 1, 150, 40]))
]
CASES += [("rows", 130, 77, 72, None), ("columns", 130, 77, 72, [64, 66])]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind,m,n,k,groups", CASES)
def test_finite_gradients_stay_finite_and_none_is_lost(kind, m, n, k, groups, device):
    args, dout = _make(kind, m, n, k, groups, m + n)
    args = {name: t.to(device) if isinstance(t, torch.Tensor) else t for name, t in args.items()}
    got = _gradients(args, dout.to(device))
    for name, (value, bound) in _wanted(args, dout.to(device)).items():
        assert value.abs().max() < 60_000, "the case itself"
        off = (got[name].double() - value).abs()
        assert (off <= bound).all(), (name, float((off / bound).nan_to_num(nan=float("inf")).max()))
        assert got[name].dtype == F16
    for name in ("a", "b"):  # one at a time: the same
        assert torch.equal(_gradients(args, dout.to(device), (name,))[name], got[name])


@pytest.mark.parametrize("device", DEVICES)
def test_the_smallest_example(device):
    a, b = torch.ones(1, 8, dtype=F16, device=device), torch.full((5, 8), 1e-3, dtype=F16, device=device)
    da = _gradients({"a": a, "b": b, "out_dtype": F32}, torch.full((1, 5), 1e5, device=device), ("a",))["a"]
    torch.testing.assert_close(da.float(), torch.full((1, 8), 500.0, device=device), rtol=2.0**-9, atol=0)
    b = torch.full((5, 8), 100.0, dtype=F16, device=device)
    da = _gradients({"a": a, "b": b, "out_dtype": F32}, torch.full((1, 5), 2e-8, device=device), ("a",))["a"]
    torch.testing.assert_close(da.float(), torch.full((1, 8), 1e-5, device=device), rtol=2.0**-9, atol=2.0**-25)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_a_gradient_that_is_no_number_stays_in_its_row_and_column(value, device):
    args, dout = _make("large", 70, 256, 64, None, 1)
    args = {name: t.to(device) if isinstance(t, torch.Tensor) else t for name, t in args.items()}
    clean = _gradients(args, dout.to(device))
    dout[3, 5] = value
    got = _gradients(args, dout.to(device))
    for name, at in (("a", 3), ("b", 5)):
        others = [i for i in range(got[name].shape[0]) if i != at]
        assert not got[name][at].isfinite().any() and torch.equal(got[name][others], clean[name][others])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dout", [0.0, 2.0**-140, 2.0**126])
def test_the_ends_of_32_bits(dout, device):
    """No factor of a row is itself zero or infinite."""
    a, b = torch.ones(2, 8, dtype=F16, device=device), torch.zeros(5, 8, dtype=F16, device=device)
    b[0, 0] = 1
    d = torch.full((2, 5), dout, device=device)
    d[1] = 1.0
    got = _gradients({"a": a, "b": b, "out_dtype": F32}, d)
    want = torch.zeros(2, 8, dtype=F16, device=device)
    want[0, 0], want[1, 0] = d[0, 0].half(), 1.0
    assert torch.equal(got["a"], want)
    assert torch.equal(got["b"], (d[0, 0].double() + 1).half().expand(5, 8).to(device))


@pytest.mark.gpu
@pytest.mark.parametrize("groups", [None, [100, 0, 1, 150, 40]])
def test_captured_and_on_several_streams(groups):
    """What the parts are taken of is found anew by every replay, and shared by no two calls."""
    names = ("a", "b", "bias")

    def make(seed, by):
        args, dout = _make("rows", 300, 512, 136, groups, seed)
        lead = () if groups is None else (len(groups),)
        args = {**args, "activation": "silu", "bias": torch.zeros(*lead, 512)}
        return {name: t.cuda() if isinstance(t, torch.Tensor) else t for name, t in args.items()}, by * dout.cuda()

    args, dout = make(1, 1.0)
    _gradients(args, dout, names)
    leaves = {name: args[name].clone().requires_grad_() for name in names}
    held = dout.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grads = torch.autograd.grad(ops.matmul(**{**args, **leaves}), tuple(leaves.values()), held)
    cases = [make(seed, by) for seed, by in ((2, 2.0**-8), (3, 2.0**8), (4, 0.0), (5, 2.0**-8))]
    alone = [_gradients(*case, names) for case in cases]
    for (fresh, d), want in zip(cases, alone):
        with torch.no_grad():
            for name in names:
                leaves[name].copy_(fresh[name])
            held.copy_(d)
        graph.replay()
        for got, name in zip(grads, names):
            assert torch.equal(got, want[name]), name
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(5):
        together = []
        for stream, case in zip(streams, cases):
            with torch.cuda.stream(stream):
                together.append(_gradients(*case, names))
        torch.cuda.synchronize()
        for got, want in zip(together, alone):
            assert all(torch.equal(got[name], want[name]) for name in names)
    assert ops.check() == 0


@pytest.mark.parametrize("device", DEVICES)
def test_the_bias_alone(device):
    args, dout = _make("large", 70, 256, 64, None, 1)
    args = {name: t.to(device) if isinstance(t, torch.Tensor) else t for name, t in args.items()} | {"bias": torch.zeros(256, device=device)}
    both, alone = _gradients(args, dout.to(device), ("a", "b", "bias")), _gradients(args, dout.to(device), ("bias",))
    assert torch.equal(alone["bias"], both["bias"])
    off = (alone["bias"].double() - dout.to(device).double().sum(0)).abs()
    assert (off <= 70 * 2.0**-24 * dout.to(device).double().abs().sum(0)).all()

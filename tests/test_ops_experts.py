"""The router's choice and rows sorted by expert on the CPU: the plain statements against the definitions in 64 bits and against
differences, and refusals."""

import math

import experts_oracle as oracle
import pytest
import torch

from lplb_b200 import ops

INF, NAN = math.inf, math.nan
SCORES = [("softmax", False), ("softmax", True), ("sigmoid", False), ("sigmoid", True)]


def logits_of(tokens, experts, seed, masked=True):
    g = torch.Generator().manual_seed(seed)
    x = 3 * torch.randn(tokens, experts, generator=g)
    x = torch.where(torch.rand(tokens, experts, generator=g) < 0.3, (x / 2).round() * 2, x)  # equal ones
    if masked and tokens > 3:
        x[torch.rand(tokens, experts, generator=g) < 0.2] = -INF
        x[1] = -INF  # nothing to choose
        x[2, 1:] = -INF  # one expert
    return x


@pytest.mark.parametrize("score,renormalize", SCORES)
@pytest.mark.parametrize("tokens,experts,topk", [(0, 4, 2), (1, 1, 1), (5, 7, 7), (9, 64, 8), (4, 200, 32)])
def test_gate(tokens, experts, topk, score, renormalize):
    x = logits_of(tokens, experts, tokens + experts)
    w, idx = ops.gate_topk(x, topk, score, renormalize, 2.5)
    want, want_idx = oracle.gate(x, topk, score, renormalize, 2.5)
    assert w.dtype == torch.float32 and idx.dtype == torch.int64 and torch.equal(idx, want_idx)
    # an exponent of up to 40 is off by 40 * 2^-24, exp by 2^-23, a sum of up to 200 by 200 * 2^-24
    torch.testing.assert_close(w.double(), want, rtol=256 * 2**-24, atol=0)


@pytest.mark.parametrize("score,renormalize", SCORES)
def test_gate_gradient(score, renormalize):
    x = logits_of(9, 33, 3)
    x.requires_grad_()
    w, idx = ops.gate_topk(x, 5, score, renormalize, 1.5)
    d = torch.randn(w.shape, generator=torch.Generator().manual_seed(1))
    (dx,) = torch.autograd.grad(w, x, d)
    want = oracle.gate_gradient(x.detach(), idx, d, score, renormalize, 1.5)
    # every term is a product of numbers of up to 1, 5 and 1.5
    torch.testing.assert_close(dx.double(), want, rtol=2**-16, atol=2**-18)
    assert torch.equal(dx[1], torch.zeros(33))


@pytest.mark.parametrize("score,renormalize", SCORES)
def test_gate_gradient_against_differences(score, renormalize):
    x = logits_of(6, 12, 5, masked=False).double()
    x += 1e-3 * torch.arange(12)  # the choice stays within the step
    d = torch.randn(6, 4, generator=torch.Generator().manual_seed(2)).double()
    value = lambda z: (oracle.gate(z, 4, score, renormalize)[0] * d).sum().item()  # noqa: E731
    idx = oracle.gate(x, 4, score, renormalize)[1]
    dx = ops.reference.gate_topk_backward_reference(x, idx, d, score, renormalize)
    h = 1e-5
    for t, e in [(0, 0), (1, 3), (2, int(idx[2, 0])), (3, int(idx[3, 3])), (5, 11)]:
        up, down = x.clone(), x.clone()
        up[t, e] += h
        down[t, e] -= h
        assert abs((value(up) - value(down)) / (2 * h) - dx[t, e].item()) < 1e-8


@pytest.mark.parametrize("score,renormalize", SCORES)
def test_gate_of_values_that_are_no_numbers(score, renormalize):
    x = torch.tensor([[1.0, NAN, 2.0, -INF], [0.0, -0.0, INF, 1.0], [-1e30, -3e38, -2e38, -INF], [-200.0, -201.0, -300.0, -INF]])
    w, idx = ops.gate_topk(x, 3, score, renormalize)
    assert idx.tolist() == [[1, 2, 0], [2, 3, 0], [0, 2, 1], [0, 1, 2]]
    want, _ = oracle.gate(x, 3, score, renormalize)
    assert torch.equal(w.isnan(), want.isnan())
    torch.testing.assert_close(w.double(), want, rtol=1e-5, atol=2.0**-149, equal_nan=True)


def test_gate_refuses():
    x = torch.randn(3, 8)
    for bad in (dict(topk=0), dict(topk=9), dict(topk=2, score="tanh")):
        with pytest.raises(ValueError, match="gate_topk"):
            ops.gate_topk(x, **bad)
    for other in (x[0], x.double(), x.int(), torch.randn(2, 0), torch.randn(2, 1025)):
        with pytest.raises(ValueError, match="gate_topk"):
            ops.gate_topk(other, 1)
    with pytest.raises(ValueError, match="topk"):
        ops.gate_topk(torch.randn(2, 64), 33)


def second_gradients(device):
    """A function of x for every operator with a gradient."""
    order = ops.expert_order(torch.tensor([[0, 1], [1, -1]], device=device), 2)
    w = torch.rand(2, 2, device=device)
    b = torch.randn(8, 8, device=device).bfloat16()
    return {
        "gate_topk": lambda x: ops.gate_topk(x[:2], 2)[0],
        "take_rows": lambda x: ops.take_rows(x[:2], order),
        "combine_rows": lambda x: ops.combine_rows(x, order, w),
        "combine_rows without weights": lambda x: ops.combine_rows(x, order),
        "matmul": lambda x: ops.matmul(x.bfloat16(), b, activation="silu"),
    }


def no_second_gradient(name, device):
    x = torch.randn(4, 8, device=device, requires_grad=True)
    y = second_gradients(device)[name](x)
    (dx,) = torch.autograd.grad((y * y).sum(), x, create_graph=True)
    want = torch.autograd.grad((y * y).sum(), x)[0]
    assert torch.equal(dx.detach(), want)
    with pytest.raises(RuntimeError, match="gradient's gradient"):
        (dx * dx).sum().backward()


@pytest.mark.parametrize("name", list(second_gradients("cpu")))
def test_no_second_gradient(name):
    no_second_gradient(name, "cpu")


def ids_of(tokens, topk, experts, seed, dtype=torch.int64):
    g = torch.Generator().manual_seed(seed)
    idx = torch.randint(-1, experts, (tokens, topk), generator=g)
    if tokens > 2:
        idx[0] = experts  # a number that no expert has
        idx[1] = 0  # the same one several times
    return idx.to(dtype)


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
@pytest.mark.parametrize("tokens,topk,experts", [(0, 2, 3), (1, 1, 1), (7, 3, 4), (33, 8, 48)])
def test_order(tokens, topk, experts, dtype):
    idx = ids_of(tokens, topk, experts, tokens, dtype)
    got = ops.expert_order(idx, experts)
    for a, b in zip(got, oracle.order(idx, experts)):
        assert a.dtype == torch.int32 and torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,topk,hidden", [(0, 2, 4), (1, 1, 1), (13, 3, 7)])
def test_rows_there_and_back(tokens, topk, hidden, dtype):
    g = torch.Generator().manual_seed(tokens)
    idx = ids_of(tokens, topk, 5, tokens)
    order = ops.expert_order(idx, 5)
    x = torch.randn(tokens, hidden, generator=g).to(dtype).requires_grad_()
    rows = ops.take_rows(x, order)
    assert torch.equal(rows, oracle.take(x.detach(), order.place))
    drows = torch.randn(rows.shape, generator=g).to(dtype)
    (dx,) = torch.autograd.grad(rows, x, drows)
    want, size = oracle.combine(drows, order.place)
    e = oracle.half_step(dtype)
    assert ((dx.double() - want).abs() <= e * want.abs() + topk * 2**-24 * size).all()
    # and with weights
    y = torch.randn(rows.shape, generator=g).to(dtype).requires_grad_()
    w = torch.rand(tokens, topk, generator=g).requires_grad_()
    out = ops.combine_rows(y, order, w)
    want, size = oracle.combine(y.detach(), order.place, w.detach())
    assert out.dtype == dtype and ((out.double() - want).abs() <= e * want.abs() + (topk + 1) * 2**-24 * size).all()
    dout = torch.randn(out.shape, generator=g).to(dtype)
    dy, dw = torch.autograd.grad(out, (y, w), dout)
    want_y, want_w, size_w = oracle.combine_gradients(dout, y.detach(), order.place, w.detach())
    assert ((dy.double() - want_y).abs() <= (e + 2**-24) * want_y.abs()).all()
    assert ((dw.double() - want_w).abs() <= hidden * 2**-23 * size_w).all()


def test_gradients_against_differences():
    g = torch.Generator().manual_seed(0)
    order = ops.expert_order(ids_of(6, 3, 4, 9), 4)
    y, w, d = torch.randn(18, 5, generator=g).double(), torch.rand(6, 3, generator=g).double(), torch.randn(6, 5, generator=g).double()
    dy, dw = ops.reference.combine_rows_backward_reference(d, y, order.place, w)
    value = lambda y, w: (oracle.combine(y, order.place, w)[0] * d).sum().item()  # noqa: E731
    for at in ((0, 0), (3, 2), (17, 4)):
        step = torch.zeros_like(y)
        step[at] = 1e-4
        assert abs((value(y + step, w) - value(y - step, w)) / 2e-4 - dy[at].item()) < 1e-9
    for at in ((0, 0), (1, 2), (5, 1)):
        step = torch.zeros_like(w)
        step[at] = 1e-4
        assert abs((value(y, w + step) - value(y, w - step)) / 2e-4 - dw[at].item()) < 1e-9


def test_rows_in_8_bits():
    order = ops.expert_order(ids_of(9, 2, 4, 1), 4)
    q, scale = ops.quantize_fp8(torch.randn(9, 256, generator=torch.Generator().manual_seed(0)))
    for t in (q, scale):
        want = oracle.take(t.view(torch.uint8), order.place)
        got = ops.take_rows(t, order)
        assert got.dtype == t.dtype and torch.equal(got.view(torch.uint8), want)


def test_what_is_masked_is_not_read():
    idx = torch.tensor([[0, -1], [-1, -1], [1, 0]])
    order = ops.expert_order(idx, 2)
    rows = torch.randn(6, 4)
    rows[3:] = NAN  # nobody's
    w = torch.rand(3, 2)
    w[0, 1] = w[1, 0] = NAN  # of choices that are none
    out = ops.combine_rows(rows, order, w)
    assert out.isfinite().all() and torch.equal(out[1], torch.zeros(4))


def test_rows_refuse():
    order = ops.expert_order(torch.tensor([[0, 1], [1, -1]]), 2)
    x, rows = torch.randn(2, 4), torch.randn(4, 4)
    for bad in (x[0], torch.randn(3, 4), torch.randn(2, 0)):
        with pytest.raises(ValueError, match="take_rows"):
            ops.take_rows(bad, order)
    for bad in (rows[0], rows[:3], rows.double(), rows.int()):
        with pytest.raises(ValueError, match="combine_rows"):
            ops.combine_rows(bad, order)
    for bad in (torch.rand(2, 3), torch.ones(2, 2, dtype=torch.int32)):
        with pytest.raises(ValueError, match="weights"):
            ops.combine_rows(rows, order, bad)
    with pytest.raises(ValueError, match="order"):
        ops.take_rows(x, ops.ExpertOrder(order.counts, order.place.long(), order.source))
    with pytest.raises(ValueError, match="order"):
        ops.combine_rows(rows, ops.ExpertOrder(order.counts, order.place, order.source[:3]))
    with pytest.raises(ValueError, match="gradient"):
        ops.take_rows(x.double().requires_grad_(), order)
    for bad in (torch.tensor([0, 1]), torch.tensor([[0.0]]), torch.zeros(2, 0, dtype=torch.int64), torch.zeros(1, 1025, dtype=torch.int64)):
        with pytest.raises(ValueError, match="expert_order"):
            ops.expert_order(bad, 2)
    for experts in (0, 1025):
        with pytest.raises(ValueError, match="expert_order"):
            ops.expert_order(torch.tensor([[0]]), experts)

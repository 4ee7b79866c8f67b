"""What one side takes the other takes as well: whole numbers, orders and counts of any strides, lengths and boundaries."""

import pytest
import torch

from lplb_b200 import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
def test_numbers_that_are_not_whole(device):
    x, idx = torch.randn(3, 8, device=device), torch.tensor([[0, 1], [2, -1]], device=device)
    for bad in (2.9, -0.5, float("nan"), float("inf"), "two", None, 2**63, 10**30, [2]):
        with pytest.raises(ValueError, match="gate_topk: topk must be a whole number"):
            ops.gate_topk(x, bad)
        with pytest.raises(ValueError, match="expert_order: n_experts must be a whole number"):
            ops.expert_order(idx, bad)
    for good in (2, 2.0, torch.tensor(2), torch.tensor(2.0)):
        assert torch.equal(ops.gate_topk(x, good)[1], ops.gate_topk(x, 2)[1])
        assert torch.equal(ops.expert_order(idx, good).place, ops.expert_order(idx, 2).place)


@pytest.mark.parametrize("device", DEVICES)
def test_orders_and_counts_of_any_strides(device):
    idx = torch.tensor([[0, 1], [2, -1], [1, 0]], device=device)
    order = ops.expert_order(idx, 3)
    apart = lambda t: torch.stack([t, torch.full_like(t, -7)], -1)[..., 0]  # noqa: E731
    other = ops.ExpertOrder(*(apart(t) for t in order))
    turned = ops.ExpertOrder(apart(order.counts), order.place.T.contiguous().T, order.source)
    assert not any(t.is_contiguous() for t in (*other, turned.counts, turned.place))
    g = torch.Generator().manual_seed(0)
    normal = lambda *shape: torch.randn(*shape, generator=g).to(device)  # noqa: E731
    x, w, b = normal(3, 16).bfloat16().requires_grad_(), normal(3, 2).requires_grad_(), normal(3, 24, 16).bfloat16()

    def run(order, weights):
        rows = ops.take_rows(x, order)
        out = ops.combine_rows(ops.matmul(rows, b, rows=order.counts), order, weights)
        return [out, *torch.autograd.grad(out.float().square().sum(), (x, w) if weights is not None else (x,))]

    for weights in (w, None):
        want = run(order, weights)
        for these in (other, turned):
            for got, right in zip(run(these, weights), want):
                assert torch.equal(got, right)


@pytest.mark.parametrize("device", DEVICES)
def test_boundaries_and_lengths(device):
    a = torch.zeros(4, 16, dtype=torch.bfloat16, device=device)
    with pytest.raises(ValueError, match="16-byte"):
        ops.matmul(a, torch.zeros(129, dtype=torch.bfloat16, device=device)[1:].view(8, 16))
    order = ops.expert_order(torch.tensor([[0]], device=device), 1)
    long = torch.zeros(1, 1, device=device).expand(1, 2**27)
    with pytest.raises(ValueError, match="too long"):
        ops.take_rows(long, order)
    with pytest.raises(ValueError, match="too long"):
        ops.combine_rows(long, order)
    many = torch.zeros(1, 1, device=device)
    with pytest.raises(ValueError, match="fewer than"):
        ops.gate_topk(many.expand(2**31, 1), 1)
    with pytest.raises(ValueError, match="fewer than"):
        ops.expert_order(many.long().expand(2**21, 1024), 1)

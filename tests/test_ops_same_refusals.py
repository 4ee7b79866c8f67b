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

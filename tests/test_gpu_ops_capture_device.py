"""A recorded call inside a capture, of tensors on another device than the current one."""

import pytest
import torch

from lplb_b200 import ops

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _refused_beside_a_living_graph(device, current):
    a = torch.randn(32, 64, device=device).to(BF16).requires_grad_()
    b = torch.randn(64, 64, device=device).to(BF16)
    with torch.cuda.device(device):
        living = ops.matmul(a, b)
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="still holds this leaf"):
            with torch.cuda.graph(graph):
                with torch.cuda.device(current):
                    ops.matmul(a, b)
    del living
    with torch.cuda.device(device):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            with torch.cuda.device(current):
                (da,) = torch.autograd.grad(ops.matmul(a, b), a, torch.ones(32, 64, dtype=BF16, device=device))
        graph.replay()
        torch.cuda.synchronize()
    assert torch.equal(da, torch.autograd.grad(ops.matmul(a, b), a, torch.ones(32, 64, dtype=BF16, device=device))[0])


def test_of_the_current_device():
    _refused_beside_a_living_graph(torch.device("cuda", 0), 0)


@pytest.mark.multigpu
def test_of_another_device():
    _refused_beside_a_living_graph(torch.device("cuda", 1), 0)

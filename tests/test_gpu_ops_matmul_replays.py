"""Captured passes of the product replayed back to back, each kernel let in while the one before still runs: the same bits every time."""

import pytest
import torch

from lplb_b200 import ops

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("m,n,k", [(8192, 4096, 64), (300, 512, 1024), (64, 512, 256)])
@pytest.mark.parametrize("activation,dtype,out_dtype", [("gelu", BF16, F32), ("silu", BF16, BF16), (None, F16, F32)])
@pytest.mark.parametrize("names", ["a bias", "a b bias"])
def test_back_to_back(m, n, k, activation, dtype, out_dtype, names):
    g = torch.Generator(device="cuda").manual_seed(m + k)
    normal = lambda *shape: torch.randn(*shape, device="cuda", generator=g)  # noqa: E731
    args = {"a": normal(m, k).to(dtype), "b": (normal(n, k) * k**-0.5).to(dtype), "bias": normal(n)}
    dout = normal(m, n).to(out_dtype)

    def step():
        leaves = {name: args[name].detach().requires_grad_() for name in names.split()}
        out = ops.matmul(**{**args, **leaves}, activation=activation, out_dtype=out_dtype)
        return [out.detach(), *torch.autograd.grad(out, tuple(leaves.values()), dout)]

    want = step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(200):
        graph.replay()
    for one, other in zip(got, want):
        assert torch.equal(one, other)
    assert ops.check() == 0

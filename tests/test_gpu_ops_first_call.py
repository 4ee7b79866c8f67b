"""The operators around and inside the experts whose very first call, forward and backward, is inside a capture (a process of its own)."""

import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

SCRIPT = """
import torch
from lplb_b200 import ops

g = torch.Generator().manual_seed(0)
made = lambda *s: torch.randn(*s, generator=g).cuda()
logits, x = made(300, 40).requires_grad_(), made(300, 128).bfloat16().requires_grad_()
w13, w2 = (made(40, 256, 128) * 0.1).bfloat16().requires_grad_(), (made(40, 64, 128) * 0.1).bfloat16().requires_grad_()
bias, residual = made(40, 64).requires_grad_(), made(1200, 64).requires_grad_()
dout = made(300, 64)

def step():
    w, idx = ops.gate_topk(logits, 4, renormalize=True)
    order = ops.expert_order(idx, 40)
    act = ops.matmul(ops.take_rows(x, order), w13, activation="swiglu", rows=order.counts)
    y = ops.matmul(act, w2, bias=bias, activation="gelu", residual=residual, rows=order.counts, out_dtype=torch.float32)
    out = ops.combine_rows(y, order, w)
    few = ops.matmul(x[:8], w13[0], activation="swiglu")
    return out.detach(), few.detach(), *torch.autograd.grad(out, (logits, x, w13, w2, bias, residual), dout)

torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    captured = step()
graph.replay()
torch.cuda.synchronize()
for a, b in zip(captured, step()):
    assert torch.equal(a, b)
assert ops.check() == 0
print("the same")
"""


def test_the_first_call_is_captured():
    run = subprocess.run([sys.executable, "-c", SCRIPT], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "the same" in run.stdout, run.stdout + run.stderr[-3000:]

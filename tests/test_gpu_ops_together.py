"""Calls of the 8-bit operators as several users make them at once: the first one inside a capture, all kernels on
several streams, two threads."""

import subprocess
import sys
import threading

import pytest
import torch

from lplb_b200 import Planner, cube, ops
from lplb_b200.models.moe import MoELayer

pytestmark = pytest.mark.gpu

FIRST = """
import torch
from lplb_b200 import ops
g = torch.Generator("cuda").manual_seed(0)
x, r = (torch.randn(20, 512, device="cuda", generator=g).bfloat16() for _ in range(2))
w = torch.randn(300, 512, device="cuda", generator=g)
w13, w2 = torch.randn(8, 256, 512, device="cuda", generator=g).bfloat16() * 0.05, torch.randn(8, 512, 128, device="cuda", generator=g).bfloat16() * 0.1
gate, idx = torch.rand(20, 8, device="cuda", generator=g).topk(2, -1)
rows = torch.tensor([3, 0, 9], dtype=torch.int32, device="cuda")
many = torch.randn(3000, 512, device="cuda", generator=g)
one = torch.ones(512, device="cuda")
def run():
    q, s, h, n = ops.rms_norm_fp8(x, one, r, return_normed=True)
    wq, ws = ops.quantize_weight_fp8(w)
    gq, gs = wq.view(torch.uint8).view(3, 100, 512).view(torch.float8_e4m3fn), ws.view(torch.uint8)[:3].view(3, 1, 4).view(torch.float8_e8m0fnu)
    out = torch.zeros(20, 100, device="cuda")
    ops.matmul_fp8(q, s, gq, gs, rows=rows, out=out, out_dtype=torch.float32)
    (a, sa), (b, sb) = ops.quantize_weight_fp8(w13), ops.quantize_weight_fp8(w2)
    return (h, n, ops.matmul_fp8(q, s, wq, ws), out, ops.matmul_fp8(*ops.quantize_fp8(many), wq, ws), ops.moe_few_tokens(x, idx, gate, w13, w2),
            ops.moe_few_tokens(q, idx, gate, a, b, x_scale=s, w13_scale=sa, w2_scale=sb))
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    captured = run()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(captured, run())) and ops.check() == 0
print("same")
"""


def test_the_first_call_of_a_process_inside_a_capture():
    run = subprocess.run([sys.executable, "-c", FIRST], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "same" in run.stdout, run.stdout + run.stderr[-3000:]


def _calls():
    g = torch.Generator("cuda").manual_seed(5)

    def rows(m, k):
        return ops.quantize_fp8(torch.randn(m, k, device="cuda", generator=g))

    def weights(*shape):
        return ops.quantize_weight_fp8(torch.randn(shape, device="cuda", generator=g))

    x = torch.randn(40, 1024, device="cuda", generator=g).bfloat16()
    gate, idx = torch.softmax(torch.randn(40, 16, device="cuda", generator=g), -1).topk(4, -1)
    w13, w2 = (torch.randn(16, *s, device="cuda", generator=g).mul(0.03).bfloat16() for s in ((1024, 1024), (1024, 512)))
    (q13, s13), (q2, s2) = ops.quantize_weight_fp8(w13), ops.quantize_weight_fp8(w2)
    few, many, grouped = (*rows(48, 2048), *weights(512, 2048)), (*rows(3000, 1024), *weights(2048, 1024)), (*rows(900, 512), *weights(6, 640, 512))
    counts = torch.tensor([100, 0, 333, 1, 400, 66], dtype=torch.int32, device="cuda")
    wide, norm = torch.randn(3000, 2048, device="cuda", generator=g).bfloat16(), torch.rand(2048, device="cuda", generator=g)
    return [
        lambda: ops.matmul_fp8(*few),
        lambda: ops.matmul_fp8(*many),
        lambda: ops.matmul_fp8(*grouped, rows=counts, out_dtype=torch.float32),
        lambda: ops.moe_few_tokens(x, idx, gate, w13, w2),
        lambda: ops.moe_few_tokens(x, idx, gate, q13, q2, w13_scale=s13, w2_scale=s2),
        lambda: ops.rms_norm_fp8(wide, norm, wide, return_normed=True)[3],
    ]


def test_all_kernels_at_once_on_several_streams():
    calls = _calls()
    planner = Planner(cube(), 16 + 16, 16, 8, device="cuda", warm_start=False)
    layer = MoELayer(planner, 1024, 512, 4, max_tokens=700, weight_dtype=torch.float8_e4m3fn)
    g = torch.Generator("cuda").manual_seed(6)
    x = torch.randn(700, 1024, device="cuda", generator=g).bfloat16()
    w, idx = torch.softmax(torch.randn(700, 16, device="cuda", generator=g), -1).topk(4, -1)
    phys = layer.route(idx, torch.zeros(1, dtype=torch.int32, device="cuda"), "static")
    calls.append(lambda: layer.forward_physical(x, phys, w))
    want = [call() for call in calls]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in calls], [[] for _ in calls]
    for i in range(12):
        for j, call in enumerate(calls):  # each call stays on its stream, in another order every time
            k = (i * 5 + j) % len(calls)
            with torch.cuda.stream(streams[k]):
                got[k].append(calls[k]())
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i, ys in enumerate(got) for y in ys)
    assert ops.check() == 0 and layer.check() == 0


def test_two_threads():
    calls = _calls()
    want = [call() for call in calls]
    torch.cuda.synchronize()
    wrong = []

    def user():
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(15):
                for i, call in enumerate(calls):
                    y = call()
                    stream.synchronize()
                    if not torch.equal(y, want[i]):
                        wrong.append(i)
            stream.synchronize()

    threads = [threading.Thread(target=user) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong and ops.check() == 0

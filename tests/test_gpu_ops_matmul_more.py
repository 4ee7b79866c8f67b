"""The product with an epilogue: waits that run out, sums in 32 bits, calls from several threads, without a graph, and beside others."""

import threading

import pytest
import torch
from test_gpu_ops_errors import TIMEOUT, short_budget
from test_ops_matmul import make_case, run

from lplb_b200 import ops

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


# ---------------------------------------------------------------------------------- waits that run out
def _ones(*shape):
    return torch.ones(*shape, dtype=BF16, device="cuda")


def few_rows():
    k = 1 << 20
    a, b = _ones(16, k), _ones(256, k)
    return lambda: (ops.matmul(a, b, out_dtype=F32) == k).all()


def many_rows():
    k = 1 << 16
    a, b = _ones(2200, k), _ones(2048, k)
    return lambda: (ops.matmul(a, b) == k).all()


def many_rows_in_32_bits():
    k = 1 << 16
    a, b = _ones(2200, k), _ones(2048, k)
    return lambda: (ops.matmul(a, b, out_dtype=F32) == k).all()


def groups():
    k = 1 << 17
    a, b, rows = _ones(610, k), _ones(3, 512, k), torch.tensor([300, 0, 300], dtype=torch.int32, device="cuda")

    def call():
        out = ops.matmul(a, b, rows=rows)
        return (out[:600] == k).all() and not out[600:].any()

    return call


def input_gradient():
    n = 1 << 16
    a, b, d = _ones(2200, 512).requires_grad_(), _ones(n, 512), _ones(2200, n)
    out = ops.matmul(a, b)
    return lambda: (torch.autograd.grad(out, a, d, retain_graph=True)[0] == n).all()


def weight_gradient():
    m = 1 << 18
    a, b, d = _ones(m, 512), _ones(512, 512).requires_grad_(), _ones(m, 512)
    out = ops.matmul(a, b)
    return lambda: (torch.autograd.grad(out, b, d, retain_graph=True)[0] == m).all()


@pytest.mark.parametrize("make", [few_rows, many_rows, many_rows_in_32_bits, groups, input_gradient, weight_gradient])
def test_a_wait_that_runs_out_ends_the_call_with_its_code(make):
    call = make()
    assert call() and ops.check() == 0
    with short_budget():
        call()
    assert ops.check() == TIMEOUT
    assert call()  # the next call is right, and does not clear it
    assert ops.check(clear=True) == TIMEOUT and ops.check() == 0
    assert call() and ops.check() == 0


# ---------------------------------------------------------------------------------- sums in 32 bits
@pytest.mark.parametrize("m", [1, 64, 300, 2500])
@pytest.mark.parametrize("k", [512, 7168, 40_000])
@pytest.mark.parametrize("activation", [None, "swiglu"])
def test_a_result_in_32_bits_is_summed_in_32_bits(m, k, activation):
    """No part of a sum is longer than 512 products in the tensor cores, which cut off what does not fit (1.6e-8 of the sum per 16 products,
    5e-7 in all); the parts are added and rounded, each addition by 2^-24 at most of a sum that is still growing."""
    g = torch.Generator(device="cuda").manual_seed(m + k)
    a = torch.randn(m, k, device="cuda", generator=g).bfloat16()
    b = (torch.randn(512, k, device="cuda", generator=g) * k**-0.5).bfloat16()
    z = a.double() @ b.double().T
    want = ops.reference._activated(z, activation)
    got = ops.matmul(a, b, activation=activation, out_dtype=F32).double()
    off = ((got - want).norm() / want.norm()).item()
    parts = k / 512
    assert off <= (2 if activation else 1) * (8e-7 + parts**0.5 * 2**-24 + 2**-21 * (activation is not None))


# ---------------------------------------------------------------------------------- other ways to call
def test_without_a_graph():
    args, dout = make_case(300, 512, 136, [100, 0, 200], "gelu", F32, True, BF16, BF16, 1, "cuda")
    want = ops.matmul(**args)
    leaves = {name: args[name].clone().requires_grad_() for name in ("a", "b", "bias", "residual")}
    with torch.no_grad():
        out = ops.matmul(**{**args, **leaves})
    assert torch.equal(out, want) and not out.requires_grad
    with torch.inference_mode():
        assert torch.equal(ops.matmul(**{**args, **leaves}), want)


def test_from_several_threads():
    cases = [make_case(m, 512, 264, groups, "silu", F32, False, BF16, BF16, m, "cuda") for m, groups in ((300, [100, 200]), (40, None), (900, None))]
    alone = [run(*case) for case in cases]
    torch.cuda.synchronize()
    failed = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    got = run(*cases[i])
                    torch.cuda.current_stream().synchronize()
                    for name, t in got.items():
                        assert torch.equal(t, alone[i][name]), name
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


def test_two_graphs_share_nothing():
    """Two captured passes, replayed at once on two streams, each with workspaces of its own."""
    cases = [make_case(400, 512, 264, [100, 0, 250, 30], "swiglu", F32, True, BF16, BF16, seed, "cuda") for seed in (1, 2)]
    alone = [run(*case) for case in cases]
    graphs, results, keep = [], [], []
    for args, dout in cases:
        leaves = {name: args[name].clone().requires_grad_() for name in ("a", "b", "bias", "residual")}
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.matmul(**{**args, **leaves})
            grads = torch.autograd.grad(out, tuple(leaves.values()), dout)
        graphs.append(graph)
        results.append({"out": out.detach(), **{"d" + name: g for name, g in zip(leaves, grads)}})
        keep.append(leaves)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for got, want in zip(results, alone):
        for name in want:
            assert torch.equal(got[name], want[name]), name


def test_an_operand_changed_before_the_backward_pass_is_noticed():
    args, dout = make_case(20, 64, 64, None, "silu", None, False, BF16, BF16, 1, "cuda")
    a = args["a"].clone().requires_grad_()
    out = ops.matmul(a, args["b"])
    with torch.no_grad():
        args["b"].mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward(dout)


@pytest.mark.parametrize("groups", [None, [40, 24]])
def test_infinities_and_what_is_no_number_stay_in_their_rows(groups):
    args, dout = make_case(64, 256, 128, groups, "relu", None, False, BF16, BF16, 3, "cuda")
    clean = ops.matmul(**args)
    args["a"][7, 3], args["a"][50, 100] = float("inf"), float("nan")
    out = ops.matmul(**args)
    rows = torch.ones(64, dtype=torch.bool, device="cuda")
    rows[7] = rows[50] = False
    assert torch.equal(out[rows], clean[rows]) and out[50].isnan().all()


def test_a_capture_beside_a_living_graph_of_a_leaf_behind_other_operators():
    """As for a leaf itself: a weight that is cast inside the capture, logits of a router's product."""
    master = torch.randn(64, 64, device="cuda", requires_grad=True)
    x = torch.randn(32, 64, device="cuda").bfloat16()
    dout = torch.ones(32, 64, device="cuda").bfloat16()
    living = master * 2
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="still holds this leaf"):
        with torch.cuda.graph(graph):
            ops.matmul(x, master.bfloat16())
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="still holds this leaf"):
        with torch.cuda.graph(graph):
            ops.gate_topk(ops.matmul(x, master.detach().bfloat16(), out_dtype=torch.float32) + master[:32], 4)
    with torch.no_grad():  # nothing is recorded
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.matmul(x, master.bfloat16())
    assert living.requires_grad
    del living
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (got,) = torch.autograd.grad(ops.matmul(x, master.bfloat16()), master, dout)
    graph.replay()
    (want,) = torch.autograd.grad(ops.matmul(x, master.bfloat16()), master, dout)
    assert torch.equal(got, want)

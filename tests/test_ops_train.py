"""The operators together, as a training step of a mixture-of-experts layer uses them behind the planner: the output and every
gradient against automatic differentiation of the layer in 64 bits."""

import pytest
import torch

from lplb_b200 import Planner, cube, ops
from lplb_b200.models import interleave_gate_up

HIDDEN, INTER, LOGICAL, TOPK = 256, 128, 32, 4


def planner_on(device):
    planner = Planner(cube(), LOGICAL + 16, LOGICAL, 8, device=device, n_nodes=1)
    planner.update_redundancy_mapping(torch.arange(LOGICAL, 0, -1).long().to(device))  # skewed: replicas are used
    return planner


def step(p, x, router, w13, w2, planner, avail, residual):
    """The layer's output on the residual stream; weights are of logical experts."""
    weights, idx = ops.gate_topk(ops.matmul(x, router, out_dtype=torch.float32), TOPK, renormalize=True)
    order = ops.expert_order(planner.run(idx, avail), planner.n_routed_experts)
    here = planner.phy2log.long()  # a replica's gradient is its original's
    act = ops.matmul(ops.take_rows(x, order), w13[here], activation="swiglu", rows=order.counts)
    y = ops.combine_rows(ops.matmul(act, w2[here], rows=order.counts), order, weights)
    return ops.matmul(y, p, residual=residual), idx


def definition(p, x, router, w13, w2, idx, residual):
    """The same in 64 bits, expert by expert, on the experts that were chosen."""
    logits = x @ router.T
    weights = torch.softmax(logits.gather(1, idx), 1)
    y = torch.zeros_like(x)
    for e in idx.unique().tolist():
        token, k = (idx == e).nonzero(as_tuple=True)
        both = (x[token] @ w13[e].T).view(len(token), -1, 2, 128)
        act = (torch.nn.functional.silu(both[:, :, 0]) * both[:, :, 1]).flatten(1)
        y = y.index_add(0, token, act @ w2[e].T * weights[token, k].unsqueeze(1))
    return y @ p.T + residual


def inputs(tokens, device):
    g = torch.Generator().manual_seed(tokens)
    normal = lambda *shape, scale=1.0: (torch.randn(*shape, generator=g) * scale).bfloat16()  # noqa: E731
    w13 = torch.stack([interleave_gate_up(normal(INTER, HIDDEN, scale=HIDDEN**-0.5), normal(INTER, HIDDEN, scale=HIDDEN**-0.5)) for _ in range(LOGICAL)])
    made = dict(
        p=normal(HIDDEN, HIDDEN, scale=HIDDEN**-0.5), x=normal(tokens, HIDDEN), router=normal(LOGICAL, HIDDEN, scale=HIDDEN**-0.5), w13=w13,
        w2=normal(LOGICAL, HIDDEN, INTER, scale=INTER**-0.5), residual=normal(tokens, HIDDEN),
    )
    return {name: t.to(device).requires_grad_() for name, t in made.items()}, normal(tokens, HIDDEN).to(device)


# Between input and output lie roundings to bfloat16 of 2^-9 of a value at most: of the activations, the experts' rows, their sum and the output;
# on the way back of as many gradients again and of the gradients through the activation.  In the norm of a whole tensor they
# add up to no more than their number: 4, and 12.  The gradient that passes the gate is a difference of numbers of about its size and
# three times theirs, so three times as far off.
BOUNDS = dict(out=4, p=12, x=36, router=36, w13=12, w2=12, residual=0)


def train(device, tokens):
    leaves, dout = inputs(tokens, device)
    planner = planner_on(device)
    avail = torch.zeros(1, dtype=torch.int32, device=device)
    out, idx = step(planner=planner, avail=avail, **leaves)
    grads = dict(zip(leaves, torch.autograd.grad(out, tuple(leaves.values()), dout)))
    wide = {name: t.detach().double().requires_grad_() for name, t in leaves.items()}
    want = definition(idx=idx, **wide)
    wanted = dict(zip(wide, torch.autograd.grad(want, tuple(wide.values()), dout.double())))
    got = {"out": out.detach(), **grads}
    for name, value in {"out": want.detach(), **wanted}.items():
        off = (got[name].double() - value).norm() / value.norm()
        assert got[name].dtype == torch.bfloat16 and off <= BOUNDS[name] * 2.0**-9, (name, float(off))
    return leaves, dout, planner, avail, out


@pytest.mark.parametrize("tokens", [1, 77])
def test_a_training_step(tokens):
    train("cpu", tokens)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 77, 1024])
def test_a_training_step_on_the_gpu(tokens):
    train("cuda", tokens)
    assert ops.check() == 0


@pytest.mark.gpu
def test_a_captured_training_step():
    """Forward and backward in one graph, replayed on other tokens: what an eager step gives."""
    leaves, dout, planner, avail, out = train("cuda", 200)
    del out

    def all_of_it():
        y, idx = step(planner=planner, avail=avail, **leaves)
        return y.detach(), idx, torch.autograd.grad(y, tuple(leaves.values()), dout)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured, chosen, grads = all_of_it()
    fresh, _ = inputs(200, "cuda")
    with torch.no_grad():
        leaves["x"].copy_(fresh["x"].flip(0))
        leaves["w2"].mul_(0.5)
    planner.invalidate_warm_start()
    graph.replay()
    torch.cuda.synchronize()
    held = captured.clone(), chosen.clone(), [g.clone() for g in grads]
    planner.invalidate_warm_start()  # the same shares again
    y, idx, now = all_of_it()
    assert torch.equal(held[1], idx)
    # which of an expert's tokens go to its replica depends on atomics in the planner, and with it the order of rows in a sum
    torch.testing.assert_close(held[0].float(), y.float(), rtol=2**-6, atol=2**-6)
    for name, a, b in zip(leaves, held[2], now):
        off = (a.double() - b.double()).norm() / b.double().norm()
        assert off <= 2 * BOUNDS[name] * 2.0**-9, name

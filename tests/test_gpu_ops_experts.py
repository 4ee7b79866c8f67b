"""The router's choice and rows sorted by expert on the GPU against their definitions in 64 bits."""

import math

import experts_oracle as oracle
import pytest
import torch
from test_ops_experts import SCORES, ids_of, logits_of, no_second_gradient, second_gradients

from lplb_b200 import Planner, cube, ops

pytestmark = pytest.mark.gpu
INF, NAN = math.inf, math.nan
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def gate_tolerance(x, experts):
    """Of a weight, relative: the exponent's rounding (its magnitude times 2^-24, here at most 64), exp (2^-22), a sum over a lane's
    share and the warp, and a few roundings around them; each may come in twice, in a score and in the sum."""
    return 2 * (64 + 4 + experts / 32 + 5 + 4) * 2**-24


@pytest.mark.parametrize("score,renormalize", SCORES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,experts,topk", [(1, 1, 1), (5, 7, 7), (33, 64, 8), (9, 65, 1), (6, 200, 32), (7, 256, 8), (4, 300, 6), (3, 1000, 9)])
def test_gate(tokens, experts, topk, score, renormalize, dtype):
    x = logits_of(tokens, experts, tokens + experts).to(dtype)
    leaf = x.cuda().requires_grad_()
    w, idx = ops.gate_topk(leaf, topk, score, renormalize, 2.5)
    want, want_idx = oracle.gate(x, topk, score, renormalize, 2.5)
    assert w.dtype == torch.float32 and torch.equal(idx.cpu(), want_idx)
    tol = gate_tolerance(x, experts)
    assert ((w.double().cpu() - want).abs() <= tol * want).all()
    d = torch.randn(w.shape, generator=torch.Generator().manual_seed(1))
    (dx,) = torch.autograd.grad(w, leaf, d.cuda())
    want_dx = oracle.gate_gradient(x, want_idx, d, score, renormalize, 2.5)
    # each is a weight times a difference of at most the largest gradient and its mean
    size = 2.5 * d.abs().amax(1, keepdim=True).double() * 2 * want_p(x, want_idx, score, renormalize)
    assert dx.dtype == dtype
    assert ((dx.double().cpu() - want_dx).abs() <= (tol + topk * 2**-23) * size + oracle.half_step(dtype) * want_dx.abs() + smallest(dtype)).all()
    # without a gradient asked for: the same
    again, again_idx = ops.gate_topk(leaf.detach(), topk, score, renormalize, 2.5)
    assert torch.equal(again, w) and torch.equal(again_idx, idx)


def smallest(dtype):
    return 2.0**-24 if dtype == torch.float16 else 2.0**-126  # half of its smallest step, or below what bf16 and float32 flush


def want_p(x, idx, score, renormalize):
    """The scores that a gradient is proportional to, in every expert's place."""
    x = x.double()
    alive = (x > -INF).any(1, keepdim=True)
    if not renormalize:
        return torch.where(alive, torch.softmax(torch.where(alive, x, torch.zeros_like(x)), 1) if score == "softmax" else torch.sigmoid(x), torch.zeros_like(x))
    w, at = oracle.gate(x, idx.shape[1], score, True)
    p = torch.zeros_like(x)
    for t in range(len(x)):
        for k, e in enumerate(at[t].tolist()):
            if e >= 0:
                p[t, e] = w[t, k]
    return p


@pytest.mark.parametrize("score,renormalize", SCORES)
def test_gate_of_values_that_are_no_numbers(score, renormalize):
    x = torch.tensor([[1.0, NAN, 2.0, -INF], [0.0, -0.0, INF, 1.0], [-1e30, -3e38, -2e38, -INF], [-200.0, -201.0, -300.0, -INF], [-INF] * 4])
    w, idx = ops.gate_topk(x.cuda(), 3, score, renormalize)
    assert idx.tolist() == [[1, 2, 0], [2, 3, 0], [0, 2, 1], [0, 1, 2], [-1, -1, -1]]
    want, _ = oracle.gate(x, 3, score, renormalize)
    assert torch.equal(w.isnan().cpu(), want.isnan())
    torch.testing.assert_close(w.double().cpu(), want, rtol=1e-4, atol=2.0**-126, equal_nan=True)  # -200 is rounded by 2^-17


def test_gate_of_rows_apart_and_transposed():
    x = torch.randn(12, 40, generator=torch.Generator().manual_seed(0)).cuda()
    whole, idx = ops.gate_topk(x[:, :17].contiguous(), 4)
    for view in (x[:, :17], x[:, :17].T.contiguous().T):
        leaf = view.detach().requires_grad_()
        w, i = ops.gate_topk(leaf, 4)
        assert torch.equal(w, whole) and torch.equal(i, idx)
        w.backward(torch.ones(1, device="cuda").expand(12, 4))
        assert leaf.grad.shape == (12, 17)
    w, i = ops.gate_topk(torch.empty(0, 17, device="cuda"), 4)
    assert w.shape == (0, 4) and i.shape == (0, 4)


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
@pytest.mark.parametrize(
    "tokens,topk,experts",
    [(0, 2, 3), (1, 1, 1), (31, 1, 1024), (33, 8, 48), (64, 8, 272), (257, 3, 5), (1023, 9, 160), (4096, 8, 272), (8192, 8, 1), (5000, 33, 1024)],
)
def test_order(tokens, topk, experts, dtype):
    idx = ids_of(tokens, topk, experts, tokens, dtype)
    got = ops.expert_order(idx.cuda(), experts)
    want = ops.reference.expert_order_reference(idx, experts)  # itself tested against the definition
    for a, b in zip(got, want):
        assert a.dtype == torch.int32 and torch.equal(a.cpu(), b)


def test_order_of_many_choices():
    g = torch.Generator(device="cuda").manual_seed(0)
    idx = torch.randint(-1, 300, (200_000, 9), device="cuda", generator=g)[:, :8]  # rows apart
    for a, b in zip(ops.expert_order(idx, 300), ops.reference.expert_order_reference(idx, 300)):
        assert torch.equal(a, b)


def off(shape, dtype, by, g, pad=0):
    """Random rows `pad` values apart, `by` values behind a 16-byte boundary."""
    rows, cols = shape
    flat = torch.randn(rows * (cols + pad) + by, generator=g).to(dtype)[by:]
    return flat, flat.view(rows, cols + pad)[:, :cols]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize(
    "tokens,topk,hidden,by,pad",
    [
        (1, 1, 1, 0, 0), (3, 2, 7, 0, 0), (5, 8, 8, 0, 0), (64, 8, 7168, 0, 0), (70, 9, 2064, 0, 8), (21, 6, 2065, 0, 0), (21, 3, 2066, 0, 0),
        (18, 33, 40, 0, 0), (19, 4, 256, 1, 0), (19, 4, 256, 2, 6), (300, 5, 96, 0, 32), (2, 2, 20000, 0, 0),
        (1, 8, 4096, 0, 0), (300, 1, 8192, 0, 0), (700, 8, 1024, 0, 0), (40, 16, 2048, 0, 0), (30, 17, 1032, 0, 8), (20, 32, 1024, 0, 0), (20, 33, 1024, 0, 0),
    ],
)
def test_rows_there_and_back(tokens, topk, hidden, by, pad, dtype):
    g = torch.Generator().manual_seed(tokens + hidden)
    idx = ids_of(tokens, topk, 12, tokens)
    order = ops.expert_order(idx.cuda(), 12)
    place = order.place.cpu()

    def on_gpu(shape):
        flat, view = off(shape, dtype, by, g, pad)
        # the storage keeps its offset from a 16-byte boundary
        there = torch.cat([torch.zeros(by, dtype=dtype), flat]).cuda()[by:]
        return view, there.as_strided(view.shape, view.stride(), there.storage_offset())

    x, gx = on_gpu((tokens, hidden))
    assert gx.data_ptr() % 16 == by * x.itemsize % 16
    gx.requires_grad_()
    rows = ops.take_rows(gx, order)
    assert rows.is_contiguous() and torch.equal(rows.detach().cpu(), oracle.take(x, place))
    d, gd = on_gpu((tokens * topk, hidden))
    (dx,) = torch.autograd.grad(rows, gx, gd)
    e = oracle.half_step(dtype)
    tiny = smallest(dtype)
    want, size = oracle.combine(d, place)
    assert dx.dtype == dtype and ((dx.double().cpu() - want).abs() <= e * want.abs() + (topk + 1) * 2**-24 * size + tiny).all()
    y, gy = on_gpu((tokens * topk, hidden))
    w = torch.randn(tokens, topk, generator=g)
    gy, gw = gy.requires_grad_(), w.cuda().requires_grad_()
    out = ops.combine_rows(gy, order, gw)
    want, size = oracle.combine(y, place, w)
    assert out.dtype == dtype and ((out.double().cpu() - want).abs() <= e * want.abs() + (topk + 1) * 2**-24 * size + tiny).all()
    dout, gdout = on_gpu((tokens, hidden))
    dy, dw = torch.autograd.grad(out, (gy, gw), gdout)
    want_y, want_w, size_w = oracle.combine_gradients(dout, y, place, w)
    assert ((dy.double().cpu() - want_y).abs() <= (e + 2**-23) * want_y.abs() + tiny).all()
    # a thread's sum has up to hidden / 256 + 16 terms behind one another, then come 5 + 8
    assert ((dw.double().cpu() - want_w).abs() <= (hidden / 256 + 32) * 2**-24 * size_w).all()
    # one gradient alone is the same one, and so are the bits of a second call
    out = ops.combine_rows(gy, order, gw)
    assert torch.equal(torch.autograd.grad(out, gy, gdout, retain_graph=True)[0], dy)
    assert torch.equal(torch.autograd.grad(out, gw, gdout)[0], dw)
    assert torch.equal(ops.combine_rows(gy.detach(), order, gw.detach()), out)


def test_rows_without_weights_and_their_gradient():
    order = ops.expert_order(ids_of(40, 4, 6, 3).cuda(), 6)
    rows = torch.randn(160, 48, device="cuda").bfloat16().requires_grad_()
    out = ops.combine_rows(rows, order)
    assert torch.equal(out, ops.combine_rows(rows.detach(), order, torch.ones(40, 4, device="cuda")))
    dout = torch.randn_like(out)
    (drows,) = torch.autograd.grad(out, rows, dout)
    assert torch.equal(drows, ops.take_rows(dout, order))


@pytest.mark.parametrize("weights_type", [torch.bfloat16, torch.float16, torch.float64])
def test_weights_of_other_types(weights_type):
    order = ops.expert_order(ids_of(40, 4, 6, 3).cuda(), 6)
    rows = torch.randn(160, 48, device="cuda").bfloat16()
    w = torch.rand(40, 4, device="cuda").to(weights_type).requires_grad_()
    out = ops.combine_rows(rows, order, w)
    assert torch.equal(out, ops.combine_rows(rows, order, w.detach().float()))
    out.sum().backward()
    assert w.grad.dtype == weights_type


def test_what_is_masked_is_not_read():
    idx = torch.tensor([[0, -1], [-1, -1], [1, 0]]).cuda()
    order = ops.expert_order(idx, 2)
    rows = torch.randn(6, 40, device="cuda")
    rows[3:] = NAN  # nobody's
    w = torch.rand(3, 2, device="cuda")
    w[0, 1] = w[1, 0] = NAN  # of choices that are none
    rows.requires_grad_()
    w.requires_grad_()
    out = ops.combine_rows(rows, order, w)
    assert out.isfinite().all() and not out[1].any()
    dout = torch.randn_like(out)
    dout[1] = NAN  # of a token without a row
    drows, dw = torch.autograd.grad(out, (rows, w), dout)
    assert drows.isfinite().all() and not drows[3:].any() and dw.isfinite().all() and not dw[1].any()


@pytest.mark.parametrize("width", [256, 255])
def test_rows_in_8_bits(width):
    order = ops.expert_order(ids_of(90, 2, 4, 1).cuda(), 4)
    q, scale = ops.quantize_fp8(torch.randn(90, width, device="cuda"))
    for t in (q, scale):
        got = ops.take_rows(t, order)
        assert got.dtype == t.dtype and torch.equal(got.view(torch.uint8).cpu(), oracle.take(t.view(torch.uint8).cpu(), order.place.cpu()))


def test_rows_sorted_for_the_product_in_8_bits():
    """The order's counts and rows are what matmul_fp8 takes."""
    experts, k, n = 6, 256, 384
    order = ops.expert_order(ids_of(50, 3, experts, 2).cuda(), experts)
    q, scale = ops.quantize_fp8(torch.randn(50, k, device="cuda"))
    b, b_scale = ops.quantize_weight_fp8(torch.randn(experts, n, k, device="cuda"))
    rows, row_scale = ops.take_rows(q, order), ops.take_rows(scale, order)
    out = ops.matmul_fp8(rows, row_scale, b, b_scale, rows=order.counts, out_dtype=torch.float32)
    want = ops.reference.matmul_fp8_reference(rows, row_scale, b, b_scale, order.counts)
    taken = int(order.counts.sum())
    torch.testing.assert_close(out[:taken], want[:taken], rtol=1e-5, atol=1e-3)


def test_offsets_behind_2_to_the_31():
    """Rows of more than 2^31 values: 4.5 GB of bytes there and back."""
    tokens, topk, hidden = 8200, 64, 4096
    idx = torch.randint(0, 16, (tokens, topk), device="cuda", generator=torch.Generator(device="cuda").manual_seed(0))
    order = ops.expert_order(idx, 16)
    x = torch.randint(-99, 99, (tokens, hidden), device="cuda", dtype=torch.int16).bfloat16()
    rows = ops.take_rows(x, order)
    assert rows.numel() > 2**31
    last = order.source[-5:].long() // topk
    assert torch.equal(rows[-5:], x[last])
    out = ops.combine_rows(rows, order)
    assert torch.equal(out, 64 * x)  # exact: 99 * 64 has 13 bits, x at most 7, their product's last six are zero


def test_on_another_stream_and_captured():
    """A forward and a backward pass on a stream of their own, then captured once and replayed on new inputs."""
    g = torch.Generator(device="cuda").manual_seed(0)
    logits = torch.randn(50, 20, device="cuda", generator=g).requires_grad_()
    x = torch.randn(50, 96, device="cuda", generator=g).bfloat16().requires_grad_()
    dout = torch.randn(50, 96, device="cuda", generator=g).bfloat16()

    def step():
        w, idx = ops.gate_topk(logits, 4, renormalize=True)
        order = ops.expert_order(idx, 20)
        out = ops.combine_rows(ops.take_rows(x, order), order, w)
        return out.detach(), order.counts, *torch.autograd.grad(out, (logits, x), dout)

    plain = step()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = step()
    torch.cuda.current_stream().wait_stream(stream)
    for a, b in zip(plain, other):
        assert torch.equal(a, b)
    del plain, other
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (1, 2):
        with torch.no_grad():
            logits.copy_(torch.randn(50, 20, device="cuda", generator=g.manual_seed(seed)))
            x.copy_(torch.randn(50, 96, device="cuda", generator=g))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_refusals():
    x = torch.randn(4, 8, device="cuda")
    for topk in (0, 9):
        with pytest.raises(ValueError, match="gate_topk"):
            ops.gate_topk(x, topk)
    for bad in (x[0], x.double(), x.int(), torch.randn(2, 1025, device="cuda")):
        with pytest.raises(ValueError, match="gate_topk"):
            ops.gate_topk(bad, 1)
    idx = torch.tensor([[0, 1], [1, -1]], device="cuda")
    for bad in (idx[0], idx.float(), idx[:, :0]):
        with pytest.raises(ValueError, match="expert_order"):
            ops.expert_order(bad, 2)
    for experts in (0, 1025):
        with pytest.raises(ValueError, match="expert_order"):
            ops.expert_order(idx, experts)
    order, rows = ops.expert_order(idx, 2), torch.randn(4, 8, device="cuda")
    for bad in (x[0], x[:3], x[:2, :0]):
        with pytest.raises(ValueError, match="take_rows"):
            ops.take_rows(bad, order)
    for bad in (rows[0], rows[:3], rows.double()):
        with pytest.raises(ValueError, match="combine_rows"):
            ops.combine_rows(bad, order)
    for bad in (torch.rand(2, 3, device="cuda"), torch.rand(2, 2), torch.ones(2, 2, dtype=torch.int32, device="cuda")):
        with pytest.raises(ValueError, match="weights"):
            ops.combine_rows(rows, order, bad)
    on_cpu = ops.ExpertOrder(*(t.cpu() for t in order))
    with pytest.raises(ValueError, match="order"):
        ops.take_rows(x[:2], on_cpu)
    with pytest.raises(ValueError, match="order"):
        ops.combine_rows(rows, ops.ExpertOrder(order.counts, order.place.long(), order.source))
    with pytest.raises(ValueError, match="gradient"):
        ops.take_rows(torch.randn(2, 8, device="cuda", dtype=torch.float64, requires_grad=True), order)


def test_an_order_that_points_elsewhere_is_not_followed():
    """Places outside the rows (an order of another batch, or no order) reach no memory."""
    x = torch.randn(2, 64, device="cuda").requires_grad_()
    place = torch.tensor([[0, 4], [1 << 30, -7]], dtype=torch.int32, device="cuda")
    order = ops.ExpertOrder(torch.zeros(2, dtype=torch.int32, device="cuda"), place, torch.tensor([0, -1, -1, -1], dtype=torch.int32, device="cuda"))
    rows = ops.take_rows(x, order)
    assert torch.equal(rows[0], x[0]) and not rows[1:].any()
    (dx,) = torch.autograd.grad(rows, x, torch.ones_like(rows))
    assert torch.equal(dx, torch.tensor([[1.0], [0.0]], device="cuda").expand(2, 64))
    w = torch.ones(2, 2, device="cuda", requires_grad=True)
    y = torch.ones(4, 64, device="cuda", requires_grad=True)
    dy, dw = torch.autograd.grad(ops.combine_rows(y, order, w), (y, w), torch.ones(2, 64, device="cuda"))
    assert dw.tolist() == [[64, 0], [0, 0]] and torch.equal(dy[0], torch.ones(64, device="cuda")) and not dy[1:].any()


@pytest.mark.parametrize("name", list(second_gradients("cpu")))
def test_no_second_gradient(name):
    no_second_gradient(name, "cuda")


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32, torch.float64, torch.bool, torch.complex64, torch.int16])
def test_rows_of_any_type(dtype):
    order = ops.expert_order(ids_of(40, 3, 5, 4).cuda(), 5)
    x = torch.randint(0, 2, (40, 9), generator=torch.Generator().manual_seed(0)).to(dtype)
    got = ops.take_rows(x.cuda(), order)
    assert got.dtype == dtype and torch.equal(got.cpu(), oracle.take(x, order.place.cpu()))


@pytest.mark.parametrize("device", ["cpu", "cuda"])
def test_no_tokens(device):
    idx = torch.empty(0, 3, dtype=torch.int64, device=device)
    order = ops.expert_order(idx, 4)
    assert order.counts.tolist() == [0] * 4 and order.source.shape == (0,)
    x = torch.empty(0, 8, device=device).requires_grad_()
    w = torch.empty(0, 3, device=device).requires_grad_()
    out = ops.combine_rows(ops.take_rows(x, order), order, w)
    dx, dw = torch.autograd.grad(out.sum(), (x, w))
    assert out.shape == dx.shape == (0, 8) and dw.shape == (0, 3)
    logits = torch.empty(0, 5, device=device).requires_grad_()
    weights, chosen = ops.gate_topk(logits, 2)
    assert chosen.shape == (0, 2) and torch.autograd.grad(weights.sum(), logits)[0].shape == (0, 5)


def test_many_choices_per_token():
    idx = ids_of(6, 1024, 40, 2).cuda()
    order = ops.expert_order(idx, 40)
    for a, b in zip(order, ops.reference.expert_order_reference(idx, 40)):
        assert torch.equal(a, b)
    x = torch.randn(6, 24, device="cuda").requires_grad_()
    rows = ops.take_rows(x, order)
    assert torch.equal(rows, ops.reference.take_rows_reference(x, order.place, order.source))
    w = torch.rand(6, 1024, device="cuda").requires_grad_()
    d = torch.randn(6, 24, device="cuda")
    dx, dw = torch.autograd.grad(ops.combine_rows(rows, order, w), (x, w), d)
    want = (w.detach().double() * (order.place >= 0)).sum(1, keepdim=True) * d.double()
    assert ((dx.double() - want).abs() <= 1026 * 2**-23 * want.abs()).all()
    want = torch.where(order.place >= 0, (d.double() * x.detach().double()).sum(1, keepdim=True), 0.0)
    size = (d.double() * x.detach().double()).abs().sum(1, keepdim=True)
    assert ((dw.double() - want).abs() <= 32 * 2**-24 * size).all()


def test_a_gate_without_a_gradient_of_its_weights():
    """A loss that hangs on the choice's weights of some tokens only, and one that hangs on none."""
    x = torch.randn(8, 16, device="cuda").requires_grad_()
    weights, idx = ops.gate_topk(x, 3)
    (dx,) = torch.autograd.grad(weights[2:4].sum(), x)
    assert not dx[:2].any() and not dx[4:].any() and dx[2:4].any()
    assert not idx.requires_grad


def test_a_gate_whose_choices_were_overwritten_has_no_gradient():
    """The planner may write the physical experts over the gate's; the gradient, which needs the gate's, is then refused, as behind
    any other write in place, and not taken of other experts."""
    planner = Planner(cube(), 48, 32, 8, device="cuda", n_nodes=1)
    planner.update_redundancy_mapping(torch.arange(32, 0, -1).long().cuda())
    avail = torch.zeros(1, dtype=torch.int32, device="cuda")
    logits = torch.randn(64, 32, device="cuda", requires_grad=True)
    weights, idx = ops.gate_topk(logits, 4)
    kept = planner.run(idx, avail, out=torch.empty_like(idx))
    torch.autograd.grad(weights.sum(), logits, retain_graph=True)
    planner.run(idx, avail, out=idx)
    assert kept.shape == idx.shape
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(weights.sum(), logits)

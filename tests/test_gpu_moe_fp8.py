"""The MoE layer with weights in 8 bits, and its passes of a few tokens."""

import pytest
import torch

from lplb_b200 import Planner, cube, ops
from lplb_b200.models.moe import MoELayer

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn


def _layer(hidden, inter, n_logical, topk, max_tokens, dtype=FP8, **kw):
    planner = Planner(cube(), n_logical + 16, n_logical, 8, device="cuda", warm_start=False)
    layer = MoELayer(planner, hidden, inter, topk, max_tokens=max_tokens, weight_dtype=dtype, **kw)
    layer.engine.set_timeout_us(1e6)
    return layer


def _inputs(tokens, hidden, n_logical, topk, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    x = torch.randn(tokens, hidden, device="cuda", generator=g).bfloat16()
    w, idx = torch.softmax(torch.randn(tokens, n_logical, device="cuda", generator=g), -1).topk(topk, -1)
    return x, idx, w


def _avail():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


def _near(y, ref):
    """Activations and results are rounded alike; a value on a border may go the other way: one e4m3 step (2**-3) of single
    activations of hundreds, and one bf16 step of a pair's result."""
    y, ref = y.float(), ref.float()
    assert (y - ref).norm() <= 2.0**-8 * ref.norm()
    assert (y - ref).abs().max() <= 2.0**-6 * ref.abs().max()


@pytest.mark.parametrize(
    "hidden,inter,n_logical,topk,tokens",
    [(256, 128, 16, 2, 200), (512, 256, 32, 2, 1), (768, 384, 16, 2, 500), (1024, 512, 32, 4, 1000), (2048, 1024, 32, 8, 3000), (1280, 128, 16, 1, 257)],
)
def test_forward_in_8_bits(hidden, inter, n_logical, topk, tokens):
    layer = _layer(hidden, inter, n_logical, topk, max(64, tokens))
    x, idx, w = _inputs(tokens, hidden, n_logical, topk)
    y = layer.forward(x, idx, w, _avail())
    assert layer.check() == 0
    _near(y, layer.reference_forward(x, idx, w))
    q, s = ops.quantize_fp8(x)
    assert torch.equal(y, layer.forward(q, idx, w, _avail(), x_scale=s))  # converted before or on the way: the same rows


def test_rows_arrive_as_they_were_converted():
    layer = _layer(512, 256, 16, 2, 64)
    x, idx, w = _inputs(40, 512, 16, 2)
    x[3, 5], x[4, 6] = float("inf"), float("nan")
    phys = layer.route(idx, _avail())
    layer.forward_physical(x, phys, w, upto=2)
    q, _ = ops.quantize_fp8(x)
    rows, meta = layer.engine.recv_x().view(torch.uint8), layer.engine.recv_meta()
    slot_of_pair = layer.engine.pair_slot()[: phys.numel()].tolist()
    pair_of_slot = {s: p for p, s in enumerate(slot_of_pair)}
    for row in range(phys.numel()):
        pair = pair_of_slot[int(meta[row]) & 0xFFFFF]
        assert torch.equal(rows[row], q.view(torch.uint8)[pair // 2])


def test_passes_in_8_bits_repeat_their_bits_and_follow_one_another():
    layer = _layer(1024, 512, 32, 4, 1000)
    batches = [_inputs(t, 1024, 32, 4, seed=t) for t in (1000, 33, 512)]
    want = []
    for x, idx, w in batches:
        want.append(layer.forward(x, idx, w, _avail()))
        torch.cuda.synchronize()
    avail = _avail()
    got = [layer.forward(x, idx, w, avail) for _ in range(6) for x, idx, w in batches]
    torch.cuda.synchronize()
    assert layer.check() == 0 and all(torch.equal(y, want[i % 3]) for i, y in enumerate(got))


@pytest.mark.parametrize("dtype", [torch.bfloat16, FP8])
def test_few_tokens_agree_with_the_whole_layer(dtype):
    layer = _layer(1024, 512, 32, 4, 100, dtype)
    for tokens in (1, 17, 64):
        x, idx, w = _inputs(tokens, 1024, 32, 4, seed=tokens)
        layer.few_tokens = False
        whole = layer.forward(x, idx, w, _avail())
        layer.few_tokens = True
        few = layer.forward(x, idx, w, _avail())
        # the whole layer rounds every pair's result to bf16 first: half a step each, weights that add up to less than one
        assert (few.float() - whole.float()).norm() <= 2.0**-7 * whole.float().norm()
        assert layer.check() == 0
    x, idx, w = _inputs(65, 1024, 32, 4)
    before = layer.engine.epoch()
    layer.forward(x, idx, w, _avail())  # one more than the two kernels take
    assert layer.engine.epoch() == before + 1


def test_few_tokens_refuse_stale_weights_and_follow_a_new_placement():
    layer = _layer(512, 256, 32, 2, 64)
    layer.few_tokens = True
    x, idx, w = _inputs(30, 512, 32, 2)
    layer.forward(x, idx, w, _avail())
    layer.planner.update_redundancy_mapping(torch.arange(32, device="cuda") ** 3 + 1)
    with pytest.raises(RuntimeError, match="place_weights"):
        layer.forward(x, idx, w, _avail())
    layer.place_weights()
    y = layer.forward(x, idx, w, _avail())
    ref = layer.reference_forward(x, idx, w).float()
    assert (y.float() - ref).norm() <= 2.0**-7 * ref.norm()


def test_what_the_layer_in_8_bits_refuses():
    layer = _layer(512, 256, 16, 2, 64)
    x, idx, w = _inputs(30, 512, 16, 2)
    phys = layer.route(idx, _avail())
    with pytest.raises(RuntimeError, match="bf16 rows only"):
        layer.forward_physical(x, phys, w, fuse_dispatch=True)
    q, s = ops.quantize_fp8(x)
    with pytest.raises(RuntimeError, match="x must be"):
        layer.forward_physical(q, phys, w)
    with pytest.raises(RuntimeError, match="x_scale must be"):
        layer.forward_physical(q, phys, w, x_scale=s[:, :2])
    with pytest.raises(RuntimeError, match="needs weights in 8 bits"):
        _layer(512, 256, 16, 2, 64, torch.bfloat16).forward_physical(q, phys, w, x_scale=s)
    with pytest.raises(ValueError, match="weight_dtype"):
        _layer(512, 256, 16, 2, 64, torch.float16)


def test_overflowing_pairs_are_dropped_and_reported():
    layer = _layer(512, 256, 16, 2, 64, capacity_rows=128)
    x, idx, w = _inputs(64, 512, 16, 2)
    layer.forward(x, idx, w, _avail())
    assert layer.check() == 0  # 128 pairs fit exactly
    tight = _layer(512, 256, 16, 4, 64, capacity_rows=128)
    x, idx, w = _inputs(64, 512, 16, 4)
    y = tight.forward(x, idx, w, _avail())
    assert tight.check() == 13 and y.isfinite().all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, FP8])
@pytest.mark.parametrize("tokens,few", [(20, True), (20, False), (300, False)])
def test_the_block_is_its_operators_one_after_the_other(tokens, few, dtype):
    hidden, inter = 512, 256
    layer = _layer(hidden, inter, 16, 2, 300, dtype)
    layer.few_tokens = few
    g = torch.Generator("cuda").manual_seed(tokens)
    x, r = (torch.randn(tokens, hidden, device="cuda", generator=g).bfloat16() for _ in range(2))
    norm = 1 + 0.2 * torch.randn(hidden, device="cuda", generator=g).bfloat16()
    router = torch.randn(16, hidden, device="cuda", generator=g) * 0.1
    w13, w2 = torch.randn(2 * 384, hidden, device="cuda", generator=g) * hidden**-0.5, torch.randn(hidden, 384, device="cuda", generator=g) * 384**-0.5
    shared = (*ops.quantize_weight_fp8(w13), *ops.quantize_weight_fp8(w2))
    y, h = layer.forward_block(x, norm, router, _avail(), residual=r, shared=shared)
    assert layer.check() == 0
    assert torch.equal(h, x + r)
    # in plain operations, rounded where the block rounds
    f = h.float()
    n = f * torch.rsqrt((f * f).mean(-1, keepdim=True) + 1e-6) * norm.float()
    q, s = ops.reference.quantize_fp8_reference(n)
    weights, idx = torch.softmax(n.bfloat16().float() @ router.T, -1).topk(2, -1)
    routed = layer.reference_forward(n.bfloat16(), idx, weights).float() if dtype != FP8 else None
    if routed is None:  # the rows in 8 bits come from the norm in 32 bits, not from its bf16 form
        held = ops.dequantize_fp8(q, s)
        routed = torch.zeros_like(f)
        for e in idx.unique().tolist():
            gate, up, down = (ops.dequantize_weight_fp8(*ops.reference.quantize_weight_fp8_reference(w)) for w in layer.logical_weights(e))
            tok, k = (idx == e).nonzero(as_tuple=True)
            act = torch.nn.functional.silu(held[tok] @ gate.T) * (held[tok] @ up.T)
            act = ops.dequantize_fp8(*ops.reference.quantize_fp8_reference(act))
            routed.index_add_(0, tok, act @ down.T * weights[tok, k].unsqueeze(1))
    both = ops.reference.matmul_fp8_reference(q, s, *shared[:2]).unflatten(-1, (-1, 2, 128))
    act = (torch.nn.functional.silu(both[:, :, 0]) * both[:, :, 1]).flatten(1)
    want = routed + ops.reference.matmul_fp8_reference(*ops.reference.quantize_fp8_reference(act), *shared[2:])
    # four roundings to bf16 (pairs, their sum, the shared product, the sum of both), half a step of 2**-8 each at most, and
    # single values on a border of 8 bits that go the other way
    assert (y.float() - want).norm() <= 5 * 2.0**-8 * want.norm()


def test_the_block_without_a_residual_or_a_shared_expert():
    layer = _layer(512, 256, 16, 2, 64)
    x = torch.randn(9, 512, device="cuda", generator=torch.Generator("cuda").manual_seed(0)).bfloat16()
    router, norm = torch.randn(16, 512, device="cuda") * 0.1, torch.ones(512, device="cuda")
    y, h = layer.forward_block(x, norm, router, _avail())
    assert h is x
    q, s, _, normed = ops.rms_norm_fp8(x, norm, return_normed=True)
    w, idx = torch.softmax(normed.float() @ router.T, -1).topk(2, -1)
    assert torch.equal(y, layer.forward(q, idx, w, _avail(), x_scale=s))

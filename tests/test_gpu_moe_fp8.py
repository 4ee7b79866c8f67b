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

"""What a pass of the MoE layer accepts: rows that start anywhere, strides, types; and the same on both sides of 64 tokens."""

import pytest
import torch

from lplb_b200 import Planner, cube, ops
from lplb_b200.models.moe import MoELayer

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn
HIDDEN, INTER, LOGICAL, TOPK = 512, 256, 16, 2


def _layer(dtype=FP8, max_tokens=200, **kw):
    planner = Planner(cube(), LOGICAL + 16, LOGICAL, 8, device="cuda", warm_start=False)
    layer = MoELayer(planner, HIDDEN, INTER, TOPK, max_tokens=max_tokens, weight_dtype=dtype, **kw)
    layer.engine.set_timeout_us(1e6)
    return layer


def _inputs(tokens, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    x = torch.randn(tokens, HIDDEN, device="cuda", generator=g).bfloat16()
    w, idx = torch.softmax(torch.randn(tokens, LOGICAL, device="cuda", generator=g), -1).topk(TOPK, -1)
    return x, idx, w


def _avail():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


def _off_by_one(x):
    """The same values from an address that is off every boundary but its type's."""
    wide = torch.zeros(x.numel() + 16, device=x.device, dtype=torch.uint8 if x.itemsize == 1 else x.dtype)
    view = wide[1 : 1 + x.numel()].view(x.shape)
    view = view.view(x.dtype) if x.itemsize == 1 else view
    view.copy_(x)
    assert view.is_contiguous() and view.data_ptr() % 16 != 0
    return view


@pytest.mark.parametrize("fuse", [False, True])
def test_rows_in_16_bits_start_anywhere(fuse):
    layer = _layer(torch.bfloat16)
    layer.fuse_dispatch = fuse
    x, idx, w = _inputs(100)
    want = layer.forward(x, idx, w, _avail())
    assert torch.equal(layer.forward(_off_by_one(x), idx, w, _avail()), want) and layer.check() == 0
    with pytest.raises(RuntimeError, match="16-byte"):  # the engine itself does not copy
        layer.engine.forward(_off_by_one(x), layer.route(idx, _avail()), w, 8)


def test_rows_in_8_bits_start_anywhere():
    layer = _layer()
    x, idx, w = _inputs(100)
    want = layer.forward(x, idx, w, _avail())
    assert torch.equal(layer.forward(_off_by_one(x), idx, w, _avail()), want)
    q, s = ops.quantize_fp8(x)
    assert torch.equal(layer.forward(_off_by_one(q), idx, w, _avail(), x_scale=_off_by_one(s)), want) and layer.check() == 0


def test_arguments_on_the_host_are_refused():
    layer = _layer()
    x, idx, w = _inputs(100)
    phys = layer.route(idx, _avail())
    q, s = ops.quantize_fp8(x)
    for args, words in (((x.cpu(), phys, w), "x must"), ((x, phys.cpu(), w), "phys_idx must"), ((x, phys, w.cpu()), "weights must")):
        with pytest.raises(RuntimeError, match=words):
            layer.forward_physical(*args)
    with pytest.raises(RuntimeError, match="x_scale must"):
        layer.forward_physical(q, phys, w, x_scale=s.cpu())


# ------------------------------------------------------------------------------------------- both sides of 64 tokens
BOTH_SIDES = pytest.mark.parametrize("tokens", [1, 64, 65])


def _few(dtype=FP8, max_tokens=200, **kw):
    layer = _layer(dtype, max_tokens, **kw)
    layer.few_tokens = True
    return layer


@BOTH_SIDES
@pytest.mark.parametrize("dtype", [torch.bfloat16, FP8])
def test_strides_and_types_of_a_pass(dtype, tokens):
    layer = _few(dtype)
    x, idx, w = _inputs(tokens)
    phys = layer.route(idx, _avail())
    want = layer.forward_physical(x, phys, w)
    across = x.t().contiguous().t()  # strided in the last dimension
    assert torch.equal(layer.forward_physical(across, phys, w), want)
    assert torch.equal(layer.forward_physical(_off_by_one(x), phys, w), want)
    for width in (HIDDEN + 64, HIDDEN + 1):  # rows apart, on and off their boundaries
        wide = torch.zeros(tokens, width, device="cuda", dtype=x.dtype)
        wide[:, :HIDDEN] = x
        assert torch.equal(layer.forward_physical(wide[:, :HIDDEN], phys, w), want)
    assert torch.equal(layer.forward_physical(x[:1].expand(tokens, -1), phys, w), layer.forward_physical(x[:1].repeat(tokens, 1), phys, w))
    assert torch.equal(layer.forward_physical(x, phys.t().contiguous().t(), w.t().contiguous().t()), want)
    assert torch.equal(layer.forward_physical(x, phys.int(), w), want)
    assert torch.equal(layer.forward_physical(x, phys.reshape(-1), w.reshape(-1)), want)
    whole = torch.ones_like(phys)
    assert torch.equal(layer.forward_physical(x, phys, whole), layer.forward_physical(x, phys, whole.float()))
    assert torch.equal(layer.forward_physical(x, phys, w.double()), layer.forward_physical(x, phys, w.double().float()))
    assert layer.check() == 0


@BOTH_SIDES
def test_strides_of_rows_in_8_bits(tokens):
    layer = _few()
    x, idx, w = _inputs(tokens)
    phys = layer.route(idx, _avail())
    q, s = ops.quantize_fp8(x)
    want = layer.forward_physical(q, phys, w, x_scale=s)
    every_second = torch.zeros(tokens, 2 * s.shape[1], dtype=torch.uint8, device="cuda")
    every_second[:, ::2] = s.view(torch.uint8)
    strided = every_second.view(torch.float8_e8m0fnu)[:, ::2]
    assert torch.equal(layer.forward_physical(q, phys, w, x_scale=strided), want)
    assert torch.equal(layer.forward_physical(_off_by_one(q), phys, w, x_scale=_off_by_one(s)), want)
    with pytest.raises(RuntimeError, match="x must be"):
        layer.forward_physical(q, phys, w)
    with pytest.raises(RuntimeError, match="x_scale must be"):
        layer.forward_physical(q, phys, w, x_scale=s[:, :2])


@BOTH_SIDES
@pytest.mark.parametrize("dtype", [torch.bfloat16, FP8])
def test_arguments_that_require_a_gradient(dtype, tokens):
    layer = _few(dtype)
    x, idx, w = _inputs(tokens)
    phys = layer.route(idx, _avail())
    want = layer.forward_physical(x, phys, w)
    y = layer.forward_physical(x.requires_grad_(), phys, w.requires_grad_())
    assert torch.equal(y, want) and not y.requires_grad


@BOTH_SIDES
def test_the_block_with_a_router_that_is_trained(tokens):
    layer = _few()
    x, _, _ = _inputs(tokens)
    norm = torch.ones(HIDDEN, device="cuda")
    router = torch.randn(LOGICAL, HIDDEN, device="cuda", generator=torch.Generator("cuda").manual_seed(3)) * 0.1
    want, _ = layer.forward_block(x, norm, router, _avail())
    y, _ = layer.forward_block(x, norm, router.clone().requires_grad_(), _avail())
    assert torch.equal(y, want)


@pytest.mark.parametrize("tokens", [33, 65])
@pytest.mark.parametrize("few", [False, True])
def test_more_tokens_than_the_layer_was_made_for(few, tokens):
    layer = _layer(max_tokens=32)
    layer.few_tokens = few
    x, idx, w = _inputs(tokens)
    with pytest.raises(RuntimeError, match="x must be contiguous .*max_tokens"):
        layer.forward_physical(x, layer.route(idx, _avail()), w)


@BOTH_SIDES
def test_a_pass_that_is_asked_to_fuse_its_dispatch(tokens):
    x, idx, w = _inputs(tokens)
    eight = _few()
    with pytest.raises(RuntimeError, match="bf16 rows only"):
        eight.forward_physical(x, eight.route(idx, _avail()), w, fuse_dispatch=True)
    eight.fuse_dispatch = True
    with pytest.raises(RuntimeError, match="bf16 rows only"):
        eight.forward_physical(x, eight.route(idx, _avail()), w)
    layer = _few(torch.bfloat16)
    phys, before = layer.route(idx, _avail()), layer.engine.epoch()
    y = layer.forward_physical(x, phys, w, fuse_dispatch=True)
    assert layer.engine.epoch() == before + 1
    layer.few_tokens = False
    assert torch.equal(layer.forward_physical(x, phys, w, fuse_dispatch=True), y)


def test_a_layer_beyond_the_short_pass_takes_the_whole_one():
    hidden = 16384 + 256
    planner = Planner(cube(), LOGICAL + 16, LOGICAL, 8, device="cuda", warm_start=False)
    layer = MoELayer(planner, hidden, 128, TOPK, max_tokens=64)
    x = torch.randn(7, hidden, device="cuda").bfloat16()
    _, idx, w = _inputs(7)
    want = layer.forward(x, idx, w, _avail(), "static")
    layer.few_tokens = True
    assert torch.equal(layer.forward(x, idx, w, _avail(), "static"), want)


def test_the_short_passes_range_is_said_alike():
    from lplb_b200 import _native
    from lplb_b200.ops import fp8

    for name in ("TOKENS", "TOPK", "EXPERTS", "HIDDEN", "INTER"):
        assert getattr(_native.load(), f"MOE_FEW_MAX_{name}") == getattr(fp8, f"MOE_FEW_MAX_{name}")

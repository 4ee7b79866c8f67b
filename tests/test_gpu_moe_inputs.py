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

"""What the dispatch in 8 bits leaves in the receive buffer: rows and their scales, and what the ranks' worker checks, on one rank."""

import pytest
import torch

from lplb_b200 import Planner, cube, ops, ring
from lplb_b200.models.moe import MoELayer
from tests.dist_fp8_worker import passes

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn


@pytest.mark.parametrize("hidden", [256, 768, 7168])
@pytest.mark.parametrize("converted", [False, True])
def test_scales_arrive_with_their_rows(converted, hidden):
    planner = Planner(cube(), 16 + 16, 16, 8, device="cuda", warm_start=False)
    layer = MoELayer(planner, hidden, 128, 2, max_tokens=64, weight_dtype=FP8)
    g = torch.Generator("cuda").manual_seed(hidden)
    blocks = torch.exp2(torch.randint(-20, 20, (40, hidden // 128, 1), device="cuda", generator=g).float())  # scales far apart
    x = (torch.randn(40, hidden // 128, 128, device="cuda", generator=g) * blocks).reshape(40, hidden).bfloat16()
    x[3, 5], x[4, 6], x[5] = float("inf"), float("nan"), 0
    w, idx = torch.softmax(torch.randn(40, 16, device="cuda", generator=g), -1).topk(2, -1)
    phys = layer.route(idx, torch.zeros(1, dtype=torch.int32, device="cuda"))
    q, s = ops.quantize_fp8(x)
    layer.engine.recv_scale().view(torch.uint8).fill_(0)
    if converted:
        layer.forward_physical(q, phys, w, upto=2, x_scale=s)
    else:
        layer.forward_physical(x, phys, w, upto=2)
    meta, slots = layer.engine.recv_meta()[: phys.numel()], layer.engine.pair_slot()[: phys.numel()].long()
    pair_of_slot = torch.empty_like(slots)
    pair_of_slot[slots] = torch.arange(phys.numel(), device="cuda")
    token = pair_of_slot[(meta & 0xFFFFF).long()] // 2
    assert torch.equal(layer.engine.recv_scale().view(torch.uint8)[: phys.numel()], s.view(torch.uint8)[token])
    assert torch.equal(layer.engine.recv_x().view(torch.uint8)[: phys.numel()], q.view(torch.uint8)[token])


def test_what_the_ranks_check_on_one_rank():
    planner = Planner(ring(2), 8 + 2, 8, 2, device="cuda", warm_start=False)
    layer = MoELayer(planner, 512, 256, 4, max_tokens=512, weight_dtype=FP8)
    layer.engine.set_timeout_us(2e5)
    passes(layer, layer, 8, rank=0)
    with pytest.raises(RuntimeError, match="no scales"):
        MoELayer(planner, 512, 256, 4, max_tokens=512).engine.recv_scale()

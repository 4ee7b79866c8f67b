"""Worker run by tests/test_multigpu_fp8.py under torch.distributed.run (one rank per GPU).

The expert-parallel layer with weights in 8 bits: rows and their scales cross to the peers, and ranks that hold their weights in
different types are refused when the layer is made.
"""

import os
import sys

import torch
import torch.distributed as dist

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from lplb_b200 import Planner, cube, ops, ring  # noqa: E402
from lplb_b200.models.moe import MoELayer  # noqa: E402

FP8 = torch.float8_e4m3fn


def passes(layer, reference, n_logical, rank, steps=4):
    """Passes of bf16 rows and of rows already in 8 bits, by both routing policies, against the plain layer."""
    for step in range(steps):
        g = torch.Generator(device=layer.device).manual_seed(1000 * step + rank)
        tokens = 300 + 17 * rank
        x = torch.randn(tokens, layer.hidden, device=layer.device, generator=g).bfloat16()
        logits = torch.randn(tokens, n_logical, device=layer.device, generator=g) + torch.linspace(-1, 1, n_logical, device=layer.device)
        w, idx = torch.softmax(logits, -1).topk(layer.topk, dim=-1)
        avail = torch.zeros(1, dtype=torch.int32, device=layer.device)
        policy = "lplb" if step % 2 == 0 else "static"
        if step < 2:
            out = layer.forward(x, idx, w, avail, policy)
        else:
            q, scale = ops.quantize_fp8(x)
            out = layer.forward(q, idx, w, avail, policy, x_scale=scale)
        torch.cuda.synchronize(layer.device)
        assert layer.check() == 0, layer.engine.status().tolist()
        want = reference.reference_forward(x, idx, w).float()
        # rounded alike; an activation on a border may go one step the other way, and pairs are rounded to bf16
        assert (out.float() - want).norm() <= 2.0**-8 * want.norm(), f"rank {rank} step {step}"
        assert (out.float() - want).abs().max() <= 2.0**-6 * want.abs().max(), f"rank {rank} step {step}"


def main():
    rank, world = int(os.environ["RANK"]), int(os.environ["WORLD_SIZE"])
    dev = torch.device("cuda", int(os.environ["LOCAL_RANK"]))
    torch.cuda.set_device(dev)
    dist.init_process_group("nccl", device_id=dev)
    group = dist.group.WORLD
    r2o = cube() if world == 8 else ring(world)
    n_logical = 4 * world
    n_routed = n_logical + r2o.shape[1] * world
    planner = Planner(r2o, n_routed, n_logical, world, group, device=dev, comm="p2p", warm_start=False)
    layer = MoELayer(planner, 512, 256, 4, max_tokens=512, group=group, capacity_factor=4.0, weight_dtype=FP8)
    layer.engine.set_timeout_us(2e5)
    alone = Planner(r2o, n_routed, n_logical, world, device=dev)
    reference = MoELayer(alone, 512, 256, 4, max_tokens=512, weight_dtype=FP8)  # its weights only
    passes(layer, reference, n_logical, rank)
    dist.barrier(group=group)
    try:
        MoELayer(planner, 512, 256, 4, max_tokens=512, group=group, weight_dtype=FP8 if rank % 2 else torch.bfloat16)
        raise AssertionError("ranks of different weight types were accepted")
    except ValueError as error:
        assert "same type" in str(error)
    dist.barrier(group=group)
    torch.cuda.synchronize(dev)
    if rank == 0:
        print("DIST_FP8_WORKER_OK", world)
    dist.destroy_process_group()


if __name__ == "__main__":
    main()

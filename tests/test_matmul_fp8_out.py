"""An output that the caller gives to matmul_fp8 counts as changed in place, as torch's own operations count it."""

import pytest
import torch

from lplb_b200 import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _operands(device, m=5):
    a, a_scale = ops.quantize_fp8(torch.randn(m, 64, device=device))
    b, b_scale = ops.quantize_weight_fp8(torch.randn(24, 64, device=device))
    return a, a_scale, b, b_scale


@pytest.mark.parametrize("m", [5, 300])
@pytest.mark.parametrize("device", DEVICES)
def test_the_outputs_version_is_raised(device, m):
    args = _operands(device, m)
    out = torch.zeros(m, 24, device=device)
    before = out._version
    assert ops.matmul_fp8(*args, out=out, out_dtype=torch.float32) is not None and out._version > before
    # a value that autograd has saved and that is overwritten is an error, not a wrong gradient
    x = torch.ones(m, 24, device=device, requires_grad=True)
    y = (x * out).sum()
    ops.matmul_fp8(*args, out=out, out_dtype=torch.float32)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    view = torch.zeros(m, 30, device=device)
    before = view._version
    ops.matmul_fp8(*args, out=view[:, 3:27], out_dtype=torch.float32)
    assert view._version > before


@pytest.mark.parametrize("device", DEVICES)
def test_an_output_that_requires_a_gradient(device):
    args = _operands(device)
    leaf = torch.zeros(5, 24, device=device, requires_grad=True)
    for out in (leaf, leaf * 1):
        with pytest.raises(ValueError, match="out requires a gradient"):
            ops.matmul_fp8(*args, out=out, out_dtype=torch.float32)
    with torch.no_grad():
        ops.matmul_fp8(*args, out=leaf, out_dtype=torch.float32)
    assert torch.equal(leaf.detach(), ops.matmul_fp8(*args, out_dtype=torch.float32))


@pytest.mark.parametrize("device", DEVICES)
def test_an_output_made_in_inference_mode(device):
    args = _operands(device)
    with torch.inference_mode():
        out = torch.zeros(5, 24, device=device)
        ops.matmul_fp8(*args, out=out, out_dtype=torch.float32)
    assert torch.equal(out, ops.matmul_fp8(*args, out_dtype=torch.float32))

"""Activations far below zero, in 32 bits: their values are small there, and right.

z is given exactly (rows of one value, a weight of ones and zeros).  gelu: the distribution's function is taken of an argument that is off by
2^-23.4 of itself, which is z^2 times that of the value, and rounded to 2^-21; silu and the slopes: e^x is good to 2 + 1.2 |x| units of
2^-23, quotient, products and sums to a few more."""

import pytest
import torch

from lplb_b200 import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
F32 = torch.float32


def _run(z, activation, device, dtype, rows=None):
    """(values, slopes) of act at z, through a product of 8 columns and its bias's gradient, a call for each value's slope."""
    a = torch.zeros(len(z), 8, dtype=dtype, device=device)
    a[:, 0] = z
    assert torch.equal(a[:, 0].double().cpu(), z.double()), "the case itself"
    b = torch.zeros(len(z), 1, 8, dtype=dtype, device=device)
    b[:, 0, 0] = 1
    bias = torch.zeros(len(z), 1, device=device).requires_grad_()
    out = ops.matmul(a, b, bias, activation, rows=torch.ones(len(z), dtype=torch.int32, device=device), out_dtype=F32)
    (slope,) = torch.autograd.grad(out.sum(), bias)
    few = torch.stack([ops.matmul(a[i : i + 1], b[i], None, activation, out_dtype=F32)[0, 0] for i in range(0, len(z), 16)])
    assert torch.equal(few, out[::16, 0])  # one row by the kernel of few rows: the same bits
    return out[:, 0].detach().double().cpu(), slope[:, 0].double().cpu()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gelu(dtype, device):
    z = torch.linspace(-12.5, 4, 400).to(dtype)
    got, slope = _run(z, "gelu", device, dtype)
    z = z.double()
    cdf, density = 0.5 * torch.special.erfc(-z * 0.5**0.5), torch.exp(-0.5 * z * z) * (2 * torch.pi) ** -0.5
    off = (z * z + 4) * 2.0**-23.4 + 2.0**-21
    assert ((got - z * cdf).abs() <= off * (z * cdf).abs()).all(), ((got - z * cdf) / (z * cdf)).abs().max()
    bound = off * cdf + (z * density).abs() * (6 + 0.6 * z * z) * 2.0**-23 + 2.0**-23 * (cdf + (z * density).abs())
    assert ((slope - cdf - z * density).abs() <= bound).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_silu(dtype, device):
    z = torch.linspace(-80, 20, 400).to(dtype)
    got, slope = _run(z, "silu", device, dtype)
    z = z.double()
    s = torch.sigmoid(z)
    off = (8 + 1.2 * z.abs()) * 2.0**-23
    assert ((got - z * s).abs() <= off * (z * s).abs()).all()
    assert ((slope - s * (1 + z * (1 - s))).abs() <= 2 * off * s * (1 + z.abs() * (1 - s))).all()

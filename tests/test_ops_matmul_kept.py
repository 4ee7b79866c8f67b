"""What the product keeps for its backward pass is kept in 32 bits, beside results in 16 bits too.

Shown by the bias's gradient in 32 bits, which is summed before dz is rounded: off by the slope's own evaluation and by what z is off.  z is a
sum of k products in 32 bits, off by (k / 16 + 32) * 2^-23 of the sum of magnitudes and half a step of itself; the slope's slope is at most 1
(a gated one's: the other factor), its evaluation good to 2^-18 (|z| + 1) up to |z| = 6 (2 + 1.2 |z| units of 2^-23 for an exponential, a few
for the rest).  A z that was rounded to 16 bits is beyond these bounds."""

import pytest
import torch
from experts_oracle import act, parts_of
from test_ops_matmul import make_case, run

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
F32, K, N = torch.float32, 64, 512
DTYPES, ACTIVATIONS = [torch.bfloat16, torch.float16], ["gelu", "silu", "swiglu"]
# one matrix of few rows; rows of whole words on boundaries; a residual off them, for which results leave another way
WAYS = {"few rows": (5, None, False), "whole words": (40, [30, 10], False), "others": (40, [30, 10], True)}


def _case(activation, dtype, way, device):
    m, groups, off = WAYS[way]
    args, dout = make_case(m, N, K, groups, activation, F32, off, dtype, dtype, 11, device)
    if off:
        wide = torch.zeros(m, args["residual"].shape[1] + 1, dtype=dtype, device=device)
        wide[:, 1:] = args["residual"]
        args["residual"] = wide[:, 1:]
    return args, dout


def _dbias(args, dout, keep=lambda z: z):
    """(dbias, bound) in 64 bits; the slopes are taken at what `keep` makes of z."""
    a, b, bias, rows, activation = args["a"].double(), args["b"].double(), args["bias"].double(), args["rows"], args["activation"]
    d, parts = dout.double(), parts_of(len(a), args["rows"])
    z, z_err = a.new_zeros(len(a), N), a.new_zeros(len(a), N)
    for e, part in parts:
        at = slice(None) if e is None else e
        z[part], z_err[part] = a[part] @ b[at].T + bias[at], (K / 16 + 32) * 2.0**-23 * (a[part].abs() @ b[at].abs().T + bias[at].abs())
    z_err += 2.0**-23 * z.abs()
    z = keep(z).requires_grad_()
    (dz,) = torch.autograd.grad(act(z, activation), z, d)
    z = z.detach()
    if activation == "swiglu":
        (gate, up), (g_err, u_err) = (t.view(len(a), -1, 2, 128).unbind(2) for t in (z, z_err))
        by = d.view(len(a), -1, 128).abs()
        to_gate = by * ((up.abs() + u_err) * (g_err + 2.0**-18 * (gate.abs() + 1)) + 1.13 * u_err)
        err = torch.stack((to_gate, by * (1.13 * g_err + 2.0**-18 * gate.abs())), 2).reshape(len(a), -1)
    else:
        err = d.abs() * (z_err + 2.0**-18 * (z.abs() + 1))
    err += 2.0**-21 * dz.abs()
    sums = lambda t: torch.stack([t[part].sum(0) for _, part in parts]).view(args["bias"].shape)  # noqa: E731
    return sums(dz), sums(err)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("activation", ACTIVATIONS)
def test_kept_in_32_bits(activation, dtype, way, device):
    args, dout = _case(activation, dtype, way, device)
    got = run(args, dout)
    assert got["out"].dtype == dtype and got["dbias"].dtype == F32
    want, bound = _dbias(args, dout)
    off = (got["dbias"].double() - want).abs()
    assert (off <= bound).all(), float((off / bound).max())


@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("activation", ACTIVATIONS)
def test_a_rounded_one_would_be_seen(activation, dtype, way):
    args, dout = _case(activation, dtype, way, "cpu")
    (want, bound), (rounded, _) = _dbias(args, dout), _dbias(args, dout, lambda z: z.to(dtype).double())
    assert ((rounded - want).abs() > bound).any()
    # or one whose low half was lost on its way
    (cut, _) = _dbias(args, dout, lambda z: (z.float().view(torch.int32) & -65536).view(F32).double())
    assert ((cut - want).abs() > bound).any()

"""The plain statements of the 8-bit operators against their definitions in 64 bits, and refusals, without a GPU."""

import math

import pytest
import torch

from lplb_b200 import ops
from lplb_b200.ops import reference

BLOCK = 128


def grid_values():
    """Every finite magnitude of e4m3, from its definition: 2**-9 steps below 2**-6, then 8 steps per power of two."""
    values = [i * 2.0**-9 for i in range(8)]
    values += [(1 + m / 8) * 2.0**e for e in range(-6, 9) for m in range(8)]
    return torch.tensor([v for v in values if v <= 448], dtype=torch.float64)


def nearest_even(v):
    """Nearest value of the grid, ties to the one with an even last digit (its index on the grid)."""
    grid = grid_values()
    a = abs(v)
    hi = int(torch.searchsorted(grid, torch.tensor(a, dtype=torch.float64)))
    hi = min(hi, len(grid) - 1)
    lo = max(hi - 1, 0)
    d_lo, d_hi = abs(a - grid[lo].item()), abs(grid[hi].item() - a)
    best = lo if d_lo < d_hi else hi if d_hi < d_lo else lo if lo % 2 == 0 else hi
    return math.copysign(grid[best].item(), v)


def by_definition(row):
    """(values on the grid, scale) of one block."""
    amax = max((abs(v) for v in row if math.isfinite(v)), default=0.0)
    s = 2.0**-126
    while amax / s > 448:
        s *= 2
    return [nearest_even(v / s) if math.isfinite(v) else math.nan for v in row], s


@pytest.mark.parametrize("scale", [1.0, 1e-30, 1e30, 2.0**-140])
@pytest.mark.parametrize("k", [1, 127, 128, 200])
def test_rows_on_the_grid(k, scale):
    g = torch.Generator().manual_seed(k)
    x = (torch.randn(3, k, generator=g) * torch.exp(3 * torch.randn(3, k, generator=g))) * scale
    q, s = ops.quantize_fp8(x)
    for r in range(3):
        for b in range(-(-k // BLOCK)):
            want, ws = by_definition(x[r, b * BLOCK : (b + 1) * BLOCK].tolist())
            assert 2.0 ** (int(s.view(torch.uint8)[r, b]) - 127) == ws
            assert q[r, b * BLOCK : (b + 1) * BLOCK].double().tolist() == want


@pytest.mark.parametrize("amax", [448.0, 448.0000305, 224.0, 256.0, 255.99998, 1.75, 1.7500001, 0.0, 3.0e38])
def test_scale_at_its_borders(amax):
    x = torch.zeros(1, 128)
    x[0, 7] = amax
    s = 2.0 ** (int(ops.quantize_fp8(x)[1].view(torch.uint8)) - 127)
    a = float(x[0, 7])
    assert a / s <= 448 and (s == 2.0**-126 or a / (s / 2) > 448)


def test_infinities_and_nan_become_nan_and_leave_their_block_alone():
    x = torch.randn(2, 256)
    clean_q, clean_s = ops.quantize_fp8(torch.where(torch.arange(256) % 50 == 0, torch.zeros(()), x))
    x[:, ::50] = torch.tensor([math.inf, -math.inf, math.nan, math.inf, math.nan, math.inf])
    q, s = ops.quantize_fp8(x)
    assert torch.equal(s.view(torch.uint8), clean_s.view(torch.uint8))
    assert q.float()[:, ::50].isnan().all()
    keep = torch.arange(256) % 50 != 0
    assert torch.equal(q.float()[:, keep], clean_q.float()[:, keep])


@pytest.mark.parametrize("shape", [(1, 1), (128, 128), (130, 300), (3, 200, 144)])
def test_weights_share_a_scale_per_block(shape):
    w = torch.randn(shape, generator=torch.Generator().manual_seed(1)) * 3
    q, s = ops.quantize_weight_fp8(w)
    assert s.shape[-2:] == (-(-shape[-2] // BLOCK), -(-shape[-1] // BLOCK))
    flat, qf, sf = (t.reshape(-1, *t.shape[-2:]) for t in (w, q.float(), s.view(torch.uint8).float()))
    for e in range(flat.shape[0]):
        for i in range(s.shape[-2]):
            for j in range(s.shape[-1]):
                part = (e, slice(i * BLOCK, (i + 1) * BLOCK), slice(j * BLOCK, (j + 1) * BLOCK))
                ws = 2.0 ** (float(sf[e, i, j]) - 127)
                assert flat[part].abs().max() / ws <= 448 < flat[part].abs().max() / (ws / 2)
                assert torch.equal(qf[part], (flat[part] / ws).to(torch.float8_e4m3fn).float())


@pytest.mark.parametrize("with_residual", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_norm_by_its_formula(dtype, with_residual):
    g = torch.Generator().manual_seed(0)
    x, r = (torch.randn(5, 300, generator=g).to(dtype) for _ in range(2))
    w = torch.randn(300, generator=g).to(dtype)
    q, s, h, normed = ops.rms_norm_fp8(x, w, r if with_residual else None, eps=1e-5, return_normed=True)
    assert torch.equal(h, (x.float() + r.float()).to(dtype) if with_residual else x)
    hd = h.double()
    n = hd / torch.sqrt(hd.square().mean(-1, keepdim=True) + 1e-5) * w.double()
    # 300 terms and three products in 32 bits: 2^-16 is over 200 half steps; then the type's own half step
    assert ((normed.double() - n).abs() <= n.abs() * (torch.finfo(dtype).eps / 2 + 2.0**-16)).all()
    scale = reference.dequantize_fp8(torch.ones_like(q.float()).to(q.dtype), s, torch.float64)
    v = reference.dequantize_fp8(q, s, torch.float64)
    assert ((v - n).abs() <= n.abs() * (2.0**-4 + 2.0**-15) + scale * 2.0**-10).all()


def test_product_of_the_values_they_stand_for():
    g = torch.Generator().manual_seed(0)
    a, sa = ops.quantize_fp8(torch.randn(7, 272, generator=g))
    b, sb = ops.quantize_weight_fp8(torch.randn(140, 272, generator=g))
    want = torch.zeros(7, 140, dtype=torch.float64)
    for k in range(272):
        col_a = a[:, k].double() * 2.0 ** (sa.view(torch.uint8)[:, k // BLOCK].double() - 127)
        row = torch.arange(140) // BLOCK
        col_b = b[:, k].double() * 2.0 ** (sb.view(torch.uint8)[row, k // BLOCK].double() - 127)
        want += col_a[:, None] * col_b[None]
    got = ops.matmul_fp8(a, sa, b, sb, out_dtype=torch.float32)
    assert (got.double() - want).abs().max() <= 272 * 2.0**-24 * want.abs().max() * 16
    assert ops.matmul_fp8(a, sa, b, sb).dtype == torch.bfloat16


def test_wrong_output_type_is_refused():
    a, sa = ops.quantize_fp8(torch.randn(2, 128))
    b, sb = ops.quantize_weight_fp8(torch.randn(4, 128))
    with pytest.raises(ValueError, match="out_dtype"):
        ops.matmul_fp8(a, sa, b, sb, out_dtype=torch.float16)

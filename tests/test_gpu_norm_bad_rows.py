"""Rows of the norm without a finite value: the scale byte is that of a block of zeros, as the plain statement and the module's
text have it, and the values are NaN."""

import pytest
import torch

from lplb_b200 import ops
from lplb_b200.ops import reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [6, 2600])  # a CTA per row, CTAs that go through the rows
@pytest.mark.parametrize("cols", [200, 256, 7168])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_scales_of_rows_with_nan_infinities_or_nothing(dtype, cols, rows):
    g = torch.Generator("cuda").manual_seed(cols)
    x = torch.randn(rows, cols, device="cuda", generator=g).to(dtype)
    x[0, 7], x[1, cols - 1], x[2, 3], x[3] = float("nan"), float("nan"), float("inf"), 0
    x[rows - 1, :130] = float("nan")
    w = torch.rand(cols, device="cuda", generator=g) + 0.5
    w[5] = -w[5]
    for eps in (1e-6, 0.0):  # without eps a row of zeros is 0 times infinity
        q, s, _ = ops.rms_norm_fp8(x, w, eps=eps)
        want_q, want_s, _ = reference.rms_norm_fp8_reference(x, w, eps=eps)
        bad = [0, 1, 2, 3, rows - 1]
        assert torch.equal(s.view(torch.uint8)[bad], want_s.view(torch.uint8)[bad])
        assert (s.view(torch.uint8)[bad] == 1).all()
        a, b = q.float()[bad], want_q.float()[bad]
        assert ((a == b) | (a.isnan() & b.isnan())).all()
        assert q.float()[[0, 1, rows - 1]].isnan().all() and (q.float()[3].isnan().all() if eps == 0 else (q.float()[3] == 0).all())
        good = torch.ones(rows, dtype=torch.bool, device="cuda")
        good[bad] = False
        # a scale on a border may go to its neighbour: the factor is rounded in another order
        assert ((s.view(torch.uint8)[good].int() - want_s.view(torch.uint8)[good].int()).abs() <= 1).all()

"""The most rows that a product takes: one more is refused, and the last of them are right."""

import pytest
import torch

from lplb_b200 import ops

MOST = 2**31 - 256


def _ones(*shape, device):
    return torch.full(shape, 0x38, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)


def _unit(*shape, device):
    return torch.full(shape, 127, dtype=torch.uint8, device=device).view(torch.float8_e8m0fnu)


@pytest.mark.parametrize("rows", [MOST + 1, 2**31 - 1, 2**31])
def test_too_many_rows_are_refused_on_the_cpu(rows):
    one = _ones(1, 16, device="cpu")
    with pytest.raises(ValueError, match="at most 2147483392 rows"):
        ops.matmul_fp8(one.expand(rows, 16), _unit(1, 1, device="cpu").expand(rows, 1), one, _unit(1, 1, device="cpu"))
    with pytest.raises(ValueError, match="at most 2147483392 rows"):
        ops.matmul_fp8(one, _unit(1, 1, device="cpu"), one.expand(rows, 16), _unit(1, 1, device="cpu").expand(-(-rows // 128), 1))


@pytest.mark.gpu
def test_the_last_rows_of_the_longest_product():
    a = torch.zeros(MOST + 1, 16, dtype=torch.uint8, device="cuda")
    a[-301:] = 0x38  # 1.0
    a[-5] = 0x40  # 2.0
    a, scale = a.view(torch.float8_e4m3fn), _unit(1, 1, device="cuda").expand(MOST + 1, 1)
    b, b_scale = _ones(1, 16, device="cuda"), _unit(1, 1, device="cuda")
    with pytest.raises(ValueError, match="at most 2147483392 rows"):
        ops.matmul_fp8(a, scale, b, b_scale)
    y = ops.matmul_fp8(a[:-1], scale[:-1], b, b_scale)
    want = torch.full((300, 1), 16.0, device="cuda", dtype=torch.bfloat16)
    want[-4] = 32.0
    assert torch.equal(y[-300:], want) and not y[-400:-300].any() and not y[:1000].any() and ops.check() == 0

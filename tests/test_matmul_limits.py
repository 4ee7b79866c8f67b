"""The most rows that the product with an epilogue takes: one more is refused, and the last of them are right."""

import pytest
import torch

from lplb_b200 import ops

MOST = 2**31 - 256


@pytest.mark.parametrize("rows", [MOST + 1, 2**31])
def test_too_many_rows_are_refused_on_the_cpu(rows):
    one = torch.ones(1, 8, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="at most 2147483392 rows"):
        ops.matmul(one.expand(rows, 8), one)


@pytest.mark.gpu
@pytest.mark.parametrize("grouped", [False, True])
def test_the_last_rows_of_the_longest_product(grouped):
    a = torch.zeros(MOST + 1, 8, dtype=torch.bfloat16, device="cuda")
    a[-301:] = 1
    a[-5] = 2
    b = torch.ones(1, 8, dtype=torch.bfloat16, device="cuda")
    more = {}
    if grouped:
        b = b.expand(2, 1, 8).contiguous()
        more["rows"] = torch.tensor([2**30 + 17, 2**31 - 1], dtype=torch.int32, device="cuda")  # what is left is the second's
    with pytest.raises(ValueError, match="at most 2147483392 rows"):
        ops.matmul(a, b, **more)
    y = ops.matmul(a[:-1], b, **more)
    want = torch.full((300, 1), 8.0, device="cuda", dtype=torch.bfloat16)
    want[-4] = 16.0
    assert torch.equal(y[-300:], want) and not y[-400:-300].any() and not y[:1000].any() and ops.check() == 0

"""Every byte that a scale can hold, by the type's definition: 2**(byte - 127), and NaN for 255."""

import math

import pytest
import torch

from lplb_b200 import ops


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_every_scale_byte_of_rows_and_weights(dtype):
    byte = torch.arange(256, dtype=torch.uint8)
    one = torch.full((256, 1), 0x38, dtype=torch.uint8).view(torch.float8_e4m3fn)  # 1.0
    rows = ops.dequantize_fp8(one, byte.view(256, 1).view(torch.float8_e8m0fnu), dtype)[:, 0].double()
    weights = ops.dequantize_weight_fp8(one.view(256, 1, 1), byte.view(256, 1, 1).view(torch.float8_e8m0fnu), dtype)[:, 0, 0].double()
    for values in (rows, weights):
        assert values[:255].tolist() == [math.ldexp(1.0, i - 127) for i in range(255)]
        assert values[255].isnan()


def test_a_product_with_a_scale_that_is_nan():
    a, a_scale = ops.quantize_fp8(torch.randn(4, 256, generator=torch.Generator().manual_seed(0)))
    b, b_scale = ops.quantize_weight_fp8(torch.randn(200, 256, generator=torch.Generator().manual_seed(1)))
    want = ops.matmul_fp8(a, a_scale, b, b_scale)
    a_scale.view(torch.uint8)[2, 1] = 255
    b_scale.view(torch.uint8)[1, 0] = 255
    y = ops.matmul_fp8(a, a_scale, b, b_scale)
    assert y[2].isnan().all() and y[:, 128:].isnan().all()
    keep = torch.tensor([0, 1, 3])
    assert torch.equal(y[keep, :128], want[keep, :128])

"""Gradients of few tiles with long sums: an input's gradient of few rows and many columns, a weight's of a small matrix and many rows."""

import pytest
import torch
from test_gpu_ops_matmul import check

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("dtype,out_dtype", [(BF16, BF16), (F16, F32)])
@pytest.mark.parametrize("m,n,k", [(64, 7168, 2048), (3, 20_000, 264), (1, 4096, 1024)])
def test_inputs(m, n, k, dtype, out_dtype):
    check(m, n, k, dtype=dtype, out_dtype=out_dtype)


@pytest.mark.parametrize("dtype,out_dtype", [(BF16, BF16), (F16, F32)])
@pytest.mark.parametrize("m,n,k", [(8192, 128, 512), (20_000, 16, 72), (40_000, 8, 8)])
def test_weights(m, n, k, dtype, out_dtype):
    check(m, n, k, bias=F32, dtype=dtype, out_dtype=out_dtype)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_weights_of_groups(dtype):
    check(30_000, 64, 128, [9, 20_000, 0, 9000, 991], "silu", bias=F32, dtype=dtype, out_dtype=dtype)

"""Products whose first CUDA call in a thread is their own: the thread has no current context then."""

import threading

import pytest
import torch

from lplb_b200 import ops

pytestmark = pytest.mark.gpu


def test_matmul_fp8_in_a_fresh_thread():
    a, a_scale = ops.quantize_fp8(torch.randn(8, 256, device="cuda"))
    b, b_scale = ops.quantize_weight_fp8(torch.randn(128, 256, device="cuda"))
    want = ops.matmul_fp8(a, a_scale, b, b_scale)
    out = torch.empty_like(want)
    stream = torch.cuda.current_stream()
    stream.synchronize()
    failed = []

    def work():
        try:
            ops.matmul_fp8(a, a_scale, b, b_scale, out=out)  # (an output that is there: nothing is allocated)
        except Exception as e:
            failed.append(e)

    thread = threading.Thread(target=work)
    thread.start()
    thread.join()
    torch.cuda.synchronize()
    assert not failed, failed
    assert torch.equal(out, want)

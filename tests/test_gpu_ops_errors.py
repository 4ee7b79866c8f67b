"""Waits inside the 8-bit operators that run out: the call ends by itself with code 21, nothing else is touched, and the next call is
right.  The budget is made so short that waits for tens of microseconds of work give up; nothing hangs and nothing is withheld."""

import contextlib

import pytest
import torch

from lplb_b200 import _native, ops

pytestmark = pytest.mark.gpu
TIMEOUT = 21


@contextlib.contextmanager
def short_budget():
    native = _native.load()
    native.set_ops_timeout_us(1e-3)
    try:
        yield
        torch.cuda.synchronize()
    finally:
        native.set_ops_timeout_us(2e6)


def _ones(*shape):
    return torch.full(shape, 0x38, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)  # 1.0


def _unit(*shape):
    return torch.full(shape, 127, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)


def few_rows():
    k = 1 << 20
    args = (_ones(16, k), _unit(16, k // 128), _ones(256, k), _unit(2, k // 128))
    return lambda: (ops.matmul_fp8(*args, out_dtype=torch.float32) == k).all()


def many_rows():
    k = 1 << 16
    args = (_ones(2048, k), _unit(2048, k // 128), _ones(2048, k), _unit(16, k // 128))
    return lambda: (ops.matmul_fp8(*args) == k).all()


def groups():
    k = 1 << 17
    rows = torch.tensor([300, 0, 300], dtype=torch.int32, device="cuda")
    args = (_ones(600, k), _unit(600, k // 128), _ones(3, 512, k), _unit(3, 4, k // 128))
    return lambda: (ops.matmul_fp8(*args, rows=rows, out_dtype=torch.float32) == k).all()


def _layer(fp8):
    tokens, experts, hidden, inter = 64, 16, 4096, 2048
    g = torch.Generator("cuda").manual_seed(0)
    x = torch.randn(tokens, hidden, device="cuda", generator=g).bfloat16()
    w13 = (torch.randn(experts, 2 * inter, hidden, device="cuda", generator=g) * hidden**-0.5).bfloat16()
    w2 = (torch.randn(experts, hidden, inter, device="cuda", generator=g) * inter**-0.5).bfloat16()
    weights, idx = torch.softmax(torch.randn(tokens, experts, device="cuda", generator=g), -1).topk(4, -1)
    scales = {}
    if fp8:
        (w13, scales["w13_scale"]), (w2, scales["w2_scale"]) = ops.quantize_weight_fp8(w13), ops.quantize_weight_fp8(w2)
    want = ops.moe_few_tokens(x, idx, weights, w13, w2, **scales)
    return lambda: (ops.moe_few_tokens(x, idx, weights, w13, w2, **scales) == want).all()


def layer_in_16_bits():
    return _layer(False)


def layer_in_8_bits():
    return _layer(True)


@pytest.mark.parametrize("make", [few_rows, many_rows, groups, layer_in_16_bits, layer_in_8_bits])
def test_a_wait_that_runs_out_ends_the_call_with_its_code(make):
    call = make()
    assert call() and ops.check() == 0
    with short_budget():
        call()
    assert ops.check() == TIMEOUT
    assert ops.check() == TIMEOUT  # it stays
    assert call()  # the next call is right, and does not clear it
    assert ops.check(clear=True) == TIMEOUT and ops.check() == 0
    assert call() and ops.check() == 0


@pytest.mark.parametrize("us", [-1.0, float("nan"), float("inf")])
def test_a_limit_that_is_none_is_refused(us):
    with pytest.raises(ValueError, match="set_ops_timeout_us"):
        _native.load().set_ops_timeout_us(us)


# ------------------------------------------------------------------------------------------- whose error it is
def _model(dtype, hidden=512, inter=256, few=False):
    from lplb_b200 import Planner, cube
    from lplb_b200.models.moe import MoELayer

    planner = Planner(cube(), 32, 16, 8, device="cuda", warm_start=False)
    layer = MoELayer(planner, hidden, inter, 4, max_tokens=128, weight_dtype=dtype)
    layer.few_tokens = few
    return layer


def _pass(layer, tokens=64):
    g = torch.Generator("cuda").manual_seed(1)
    x = torch.randn(tokens, layer.hidden, device="cuda", generator=g).bfloat16()
    w, idx = torch.softmax(torch.randn(tokens, 16, device="cuda", generator=g), -1).topk(4, -1)
    return layer.forward(x, idx, w, torch.zeros(1, dtype=torch.int32, device="cuda"), "static")


def test_a_layer_does_not_report_the_errors_of_other_calls():
    layers = [_model(torch.bfloat16), _model(torch.float8_e4m3fn, few=True)]
    for layer in layers:
        _pass(layer)
    call = few_rows()
    with short_budget():
        call()
    assert [layer.check() for layer in layers] == [0, 0]
    assert ops.check(clear=True) == TIMEOUT


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_a_layers_own_error_is_its_own_and_reset_removes_it(dtype):
    layer, other = _model(dtype, 4096, 2048, few=True), _model(dtype, few=True)
    want = _pass(layer)
    assert layer.check() == 0
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with short_budget(), torch.cuda.stream(side):
        _pass(layer)
    assert layer.check() == TIMEOUT and other.check() == 0 and ops.check() == 0
    layer.reset()
    assert layer.check() == 0
    assert torch.equal(_pass(layer), want) and layer.check() == 0


def test_the_shared_experts_errors_are_the_layers():
    layer = _model(torch.float8_e4m3fn)
    hidden, g = layer.hidden, torch.Generator("cuda").manual_seed(2)
    x = torch.randn(5, hidden, device="cuda", generator=g).bfloat16()
    norm, router = torch.ones(hidden, device="cuda"), torch.randn(16, hidden, device="cuda", generator=g) * 0.1
    shared = (*ops.quantize_weight_fp8(torch.randn(512, hidden, device="cuda")), *ops.quantize_weight_fp8(torch.randn(hidden, 256, device="cuda")))
    avail = torch.zeros(1, dtype=torch.int32, device="cuda")
    layer.forward_block(x, norm, router, avail, shared=shared)
    assert layer.check() == 0
    with short_budget():
        layer.forward_block(x, norm, router, avail, shared=shared)
    assert layer.check() == TIMEOUT and ops.check() == 0
    layer.reset()
    assert layer.check() == 0


def test_a_status_of_the_caller_takes_the_error():
    call, k = few_rows(), 1 << 20
    status = torch.zeros(4, dtype=torch.int32, device="cuda")
    args = (_ones(16, k), _unit(16, k // 128), _ones(256, k), _unit(2, k // 128))
    with short_budget():
        ops.matmul_fp8(*args, out_dtype=torch.float32, status=status)
    assert status.tolist() == [TIMEOUT, 0, 0, 0] and ops.check() == 0
    assert call()
    for bad in (status.cpu(), status.long(), status[:0]):
        with pytest.raises(ValueError, match="status must"):
            ops.matmul_fp8(*args, status=bad)

"""Arguments that the kernels refuse are refused by the plain statements too, as ValueError: types, and tensors of several devices
(the second device is `meta`, so no GPU is needed)."""

import pytest
import torch

from lplb_b200 import ops

E8M0 = torch.float8_e8m0fnu


def _product():
    a, a_scale = ops.quantize_fp8(torch.randn(3, 256))
    b, b_scale = ops.quantize_weight_fp8(torch.randn(40, 256))
    return dict(a=a, a_scale=a_scale, b=b, b_scale=b_scale)


def _layer(fp8):
    x, w = torch.randn(3, 256).bfloat16(), torch.rand(3, 2)
    w13, w2 = torch.randn(4, 256, 256).bfloat16(), torch.randn(4, 256, 128).bfloat16()
    args = dict(x=x, idx=torch.tensor([[0, 1], [2, 3], [1, 3]]), weights=w, w13=w13, w2=w2)
    if fp8:
        args["w13"], args["w13_scale"] = ops.quantize_weight_fp8(w13)
        args["w2"], args["w2_scale"] = ops.quantize_weight_fp8(w2)
        args["x"], args["x_scale"] = ops.quantize_fp8(x)
    return args


@pytest.mark.parametrize("dtype", [torch.float64, torch.int32, torch.float8_e4m3fn])
def test_types_of_weights_and_rows(dtype):
    for call, who in ((ops.quantize_weight_fp8, "quantize_weight_fp8"), (ops.quantize_fp8, "quantize_fp8")):
        with pytest.raises(ValueError, match=f"{who}.*float32, bfloat16 or float16"):
            call(torch.zeros(4, 16).to(dtype))


@pytest.mark.parametrize("name", ["a_scale", "b", "b_scale", "rows", "out"])
def test_products_over_two_devices(name):
    args = _product()
    if name == "rows":
        args.update(b=args["b"][None], b_scale=args["b_scale"][None], rows=torch.tensor([3], dtype=torch.int32))
    if name == "out":
        args.update(out=torch.zeros(3, 40), out_dtype=torch.float32)
    ops.matmul_fp8(**args)
    args[name] = args[name].to("meta")
    with pytest.raises(ValueError, match="one device"):
        ops.matmul_fp8(**args)


@pytest.mark.parametrize("name", ["weight", "residual"])
def test_norms_over_two_devices(name):
    args = dict(x=torch.randn(2, 64), weight=torch.ones(64), residual=torch.randn(2, 64))
    ops.rms_norm_fp8(**args)
    args[name] = args[name].to("meta")
    with pytest.raises(ValueError, match="one device"):
        ops.rms_norm_fp8(**args)


@pytest.mark.parametrize("fp8", [False, True])
def test_layers_over_two_devices_and_scales_of_another_type(fp8):
    args = _layer(fp8)
    ops.moe_few_tokens(**args)
    for name in args:
        if name != "x":
            with pytest.raises(ValueError, match="one device"):
                ops.moe_few_tokens(**{**args, name: args[name].to("meta")})
        if name.endswith("scale"):
            with pytest.raises(ValueError, match="float8_e8m0fnu"):
                ops.moe_few_tokens(**{**args, name: args[name].view(torch.uint8)})

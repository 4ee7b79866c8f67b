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


def _weights(n, k, groups=None):
    shape = (n, k) if groups is None else (groups, n, k)
    return ops.quantize_weight_fp8(torch.randn(shape, generator=torch.Generator().manual_seed(3)))


def test_groups_take_their_own_matrix_and_leave_the_rest():
    a, sa = ops.quantize_fp8(torch.randn(9, 144, generator=torch.Generator().manual_seed(2)))
    b, sb = _weights(20, 144, 3)
    out = torch.full((9, 20), 7.0)
    ops.matmul_fp8(a, sa, b, sb, rows=torch.tensor([2, 0, 4], dtype=torch.int32), out=out, out_dtype=torch.float32)
    for e, part in ((0, slice(0, 2)), (2, slice(2, 6))):
        want = ops.matmul_fp8(a[part], sa[part], b[e], sb[e], out_dtype=torch.float32)
        assert torch.equal(out[part], want)
    assert (out[6:] == 7).all()


@pytest.mark.parametrize(
    "change,words",
    [
        (dict(k=17), "multiple of 16"), (dict(b_k=272), "same k"), (dict(a_scale=(3, 1)), "a_scale"), (dict(b_scale=(2, 2)), "b_scale"),
        (dict(out=(3, 30)), "out must"), (dict(rows=4), "rows must|b must"), (dict(a_type=torch.float32), "a must"),
    ],
)
def test_products_that_are_refused(change, words):
    k = change.get("k", 256)
    a = torch.zeros(3, k).to(change.get("a_type", torch.float8_e4m3fn))
    b = torch.zeros(40, change.get("b_k", k)).to(torch.float8_e4m3fn)
    e8m0 = torch.float8_e8m0fnu
    a_scale = torch.ones(change.get("a_scale", (3, -(-k // 128)))).to(e8m0)
    b_scale = torch.ones(change.get("b_scale", (1, -(-k // 128)))).to(e8m0)
    rows = torch.zeros(change["rows"], dtype=torch.int32) if "rows" in change else None
    out = torch.zeros(change["out"]) if "out" in change else None
    with pytest.raises(ValueError, match=words):
        ops.matmul_fp8(a, a_scale, b, b_scale, rows=rows, out=out, out_dtype=torch.float32)


def test_rows_that_are_refused():
    with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
        ops.quantize_fp8(torch.zeros(2, 4, dtype=torch.float64))
    with pytest.raises(ValueError, match="1 to 16384"):
        ops.quantize_fp8(torch.zeros(2, 16385))
    with pytest.raises(ValueError, match="gradient"):
        ops.quantize_fp8(torch.zeros(2, 4, requires_grad=True))
    with pytest.raises(ValueError, match="weight must have"):
        ops.rms_norm_fp8(torch.zeros(2, 4), torch.ones(5))
    with pytest.raises(ValueError, match="residual must have"):
        ops.rms_norm_fp8(torch.zeros(2, 4), torch.ones(4), torch.zeros(2, 4).half())


def _layer(tokens=3, topk=2, experts=4, hidden=256, inter=128, fp8=True):
    g = torch.Generator().manual_seed(5)
    x = torch.randn(tokens, hidden, generator=g).bfloat16()
    idx = torch.stack([torch.randperm(experts, generator=g)[:topk] for _ in range(tokens)])
    w = torch.rand(tokens, topk, generator=g)
    w13 = torch.randn(experts, 2 * inter, hidden, generator=g).mul(hidden**-0.5).bfloat16()
    w2 = torch.randn(experts, hidden, inter, generator=g).mul(inter**-0.5).bfloat16()
    scales = {}
    if fp8:
        (w13, scales["w13_scale"]), (w2, scales["w2_scale"]) = ops.quantize_weight_fp8(w13), ops.quantize_weight_fp8(w2)
    return x, idx, w, w13, w2, scales


@pytest.mark.parametrize("fp8", [False, True])
def test_layer_pair_by_pair(fp8):
    x, idx, w, w13, w2, scales = _layer(fp8=fp8)
    y = ops.moe_few_tokens(x, idx, w, w13, w2, **scales).double()
    d = torch.float64
    if fp8:
        xv = reference.dequantize_fp8(*ops.quantize_fp8(x), d)
        w13, w2 = (reference.dequantize_weight_fp8(q, s, d) for q, s in ((w13, scales["w13_scale"]), (w2, scales["w2_scale"])))
    else:
        xv, w13, w2 = x.double(), w13.double(), w2.double()
    want = torch.zeros_like(y)
    for t in range(3):
        for k in range(2):
            e = int(idx[t, k])
            gate, up = w13[e, :128] @ xv[t], w13[e, 128:] @ xv[t]
            act = gate / (1 + torch.exp(-gate)) * up
            act = reference.dequantize_fp8(*reference.quantize_fp8_reference(act), d) if fp8 else act.bfloat16().double()
            want[t] += w[t, k].double() * (w2[e] @ act)
    # both round the activations; a value on a border may go either way: one step of one in 128
    step = 2.0**-3 if fp8 else 2.0**-7
    assert ((y - want).abs() <= want.abs() * 2.0**-8 + 2.0**-12 + step / 128 * want.abs().max()).all()


def test_choices_that_choose_nothing_and_choices_made_twice():
    x, idx, w, w13, w2, scales = _layer()
    idx = torch.tensor([[-1, -1], [1, 1], [9, 2]])
    y = ops.moe_few_tokens(x, idx, w, w13, w2, **scales)
    assert (y[0] == 0).all()
    once = ops.moe_few_tokens(x[1:2], idx[1:2, :1], w[1:2].sum(1, keepdim=True), w13, w2, **scales)
    assert (y[1:2].float() - once.float()).abs().max() <= 2.0**-7 * once.float().abs().max()
    assert torch.equal(y[2:], ops.moe_few_tokens(x[2:], idx[2:, 1:], w[2:, 1:], w13, w2, **scales))


@pytest.mark.parametrize(
    "change,words",
    [
        (dict(tokens=65), "at most 64"), (dict(hidden=384), "multiple of 256"), (dict(inter=64), "of 128"), (dict(idx=(3, 33)), "1 to 32"),
        (dict(weights=(3, 3)), "idx's shape"), (dict(drop="w2_scale"), "come together"), (dict(x=torch.float16), "x must be"),
        (dict(x_scale=True), "float8_e4m3fn with"),
    ],
)
def test_layers_that_are_refused(change, words):
    hidden, inter, tokens = change.get("hidden", 256), change.get("inter", 128), change.get("tokens", 3)
    x = torch.zeros(tokens, hidden, dtype=change.get("x", torch.bfloat16))
    idx = torch.zeros(change.get("idx", (tokens, 2)), dtype=torch.int64)
    w = torch.zeros(change.get("weights", tuple(idx.shape)))
    w13, w2 = torch.zeros(4, 2 * inter, hidden).to(torch.float8_e4m3fn), torch.zeros(4, hidden, inter).to(torch.float8_e4m3fn)
    kw = {n: torch.ones(4, -(-v.shape[1] // 128), -(-v.shape[2] // 128)).to(torch.float8_e8m0fnu) for n, v in (("w13_scale", w13), ("w2_scale", w2))}
    kw.pop(change.get("drop"), None)
    if "x_scale" in change:
        kw["x_scale"] = torch.ones(tokens, hidden // 128).to(torch.float8_e8m0fnu)
    with pytest.raises(ValueError, match=words):
        ops.moe_few_tokens(x, idx, w, w13, w2, **kw)


def test_kernels_of_these_operators_wait_before_they_touch_memory():
    """They start while their predecessor runs out (the launches' text, as for the layer's kernels)."""
    import re
    from pathlib import Path

    csrc = Path(__file__).resolve().parents[1] / "lplb_b200" / "csrc"
    access = re.compile(r"\batomic\w+\(|\b(tma_load|tma_gather)\w*\(|__ldc?g\(|load_raw<|ld_acquire\w*\(")
    for file, kernels in (
        ("norm_fp8.cu", ("row_fp8_kernel", "row_stream_fp8_kernel", "weight_fp8_kernel")),
        ("matmul_fp8.cuh", ("few_rows_kernel",)), ("moe_few.cuh", ("moe_few_kernel", "moe_few_plan_kernel")),
    ):
        text = re.sub(r"//[^\n]*", "", (csrc / file).read_text())
        for kernel in kernels:
            start = re.search(r"__global__[^;{]*?\b%s\([^;{]*\{" % kernel, text, re.S)
            assert start, kernel
            before = text[start.end() : text.index("wait_predecessors();", start.end())]
            assert "__global__" not in before and access.search(before) is None, kernel

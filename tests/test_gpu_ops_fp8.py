"""The kernels of the 8-bit operators against plain statements in 64 bits.

Bounds count roundings.  A sum of n products in 32 bits, in whatever order, is off by at most about n half steps of
the magnitudes' sum; the tensor core adds 32 (8 bits) or 16 (bf16) products at a time and may cut where it could round,
so ``_sum_bound`` takes a whole step (2**-23) per addition and eight more.  A result's own rounding is half a step of its type."""

import pytest
import torch

from lplb_b200 import ops
from lplb_b200.ops import reference

pytestmark = pytest.mark.gpu
D = torch.float64
HALF = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}


def _gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def _bits(t):
    return t.view(torch.uint8)


def _sum_bound(k, per):
    return (-(-k // per) + 8) * 2.0**-23


def _same_values(a, b):
    a, b = a.float(), b.float()
    return bool(((a == b) | (a.isnan() & b.isnan())).all())


# ------------------------------------------------------------------------------------------- rows in 8 bits
ROWS = [(1, 1), (1, 16), (3, 127), (2, 128), (5, 129), (64, 7168), (700, 2064), (2500, 272), (2400, 515), (3, 16384), (2400, 7168)]


@pytest.mark.parametrize("rows,cols", ROWS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_rows_have_the_plain_forms_bits(dtype, rows, cols):
    g = _gen(rows)
    x = (torch.randn(rows, cols, device="cuda", generator=g) * torch.exp(2 * torch.randn(cols, device="cuda", generator=g))).to(dtype)
    x[0, : cols // 2] = 0
    if rows > 2:
        x[1, cols // 3], x[2, cols // 2], x[2, 0] = float("inf"), float("nan"), -float("inf")
    q, s = ops.quantize_fp8(x)
    want_q, want_s = reference.quantize_fp8_reference(x)
    assert torch.equal(_bits(s), _bits(want_s))
    assert _same_values(q, want_q)


@pytest.mark.parametrize("shape", [(1, 16), (128, 128), (130, 300), (3, 257, 144), (2, 256, 7168)])
def test_weights_have_the_plain_forms_bits(shape):
    w = torch.randn(shape, device="cuda", generator=_gen(0)).bfloat16()
    q, s = ops.quantize_weight_fp8(w)
    want_q, want_s = reference.quantize_weight_fp8_reference(w)
    assert torch.equal(_bits(s), _bits(want_s)) and _same_values(q, want_q)


def _check_norm(x, w, r, eps, got):
    q, s, h, normed = got
    assert _same_values(h, x if r is None else (x.double() + r.double()).to(x.dtype))
    hd = h.double()
    n = hd / torch.sqrt(hd.square().mean(-1, keepdim=True) + eps) * w.double()
    # the sum of squares adds up at most cols / 32 terms per thread and lane, the factor and two products follow
    off = (x.shape[-1] / 32 + 16) * 2.0**-24
    # (below the smallest normal number a type's steps stay as wide as there: float16 has a step of 2**-24 below 2**-14)
    low = torch.finfo(x.dtype).smallest_normal * HALF[x.dtype]
    assert ((normed.double() - n).abs() <= n.abs() * (HALF[x.dtype] + off) + low).all()
    one = torch.ones_like(q.float()).to(torch.float8_e4m3fn)
    scale = reference.dequantize_fp8(one, s, D)
    v = reference.dequantize_fp8(q, s, D)
    assert ((v - n).abs() <= n.abs() * (2.0**-4 + off) + scale * 2.0**-10).all()
    # the smallest power of two that holds the block's largest value, or a neighbour where that is on the border
    blocks = torch.nn.functional.pad(n, (0, -n.shape[-1] % 128)).unflatten(-1, (-1, 128)).abs().amax(-1)
    first = scale[..., ::128]
    assert (blocks * (1 - 2 * off) <= 448 * first).all()
    assert ((blocks * (1 + 2 * off) > 224 * first) | (first == 2.0**-126)).all()


@pytest.mark.parametrize("with_residual", [False, True])
@pytest.mark.parametrize("rows,cols", ROWS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_norm(dtype, rows, cols, with_residual):
    g = _gen(cols)
    x, r = (torch.randn(rows, cols, device="cuda", generator=g).to(dtype) for _ in range(2))
    w = (1 + 0.3 * torch.randn(cols, device="cuda", generator=g)).to(dtype)
    r = r if with_residual else None
    _check_norm(x, w, r, 1e-5, ops.rms_norm_fp8(x, w, r, eps=1e-5, return_normed=True))


@pytest.mark.parametrize("rows", [5, 2500])
@pytest.mark.parametrize("cols,start,stride", [(256, 0, 272), (256, 8, 272), (256, 1, 259), (250, 3, 512)])
def test_norm_of_rows_apart_and_off_their_boundaries(rows, cols, start, stride):
    g = _gen(1)
    wide = torch.randn(2, rows, stride, device="cuda", generator=g).bfloat16()
    x, r = wide[0, :, start : start + cols], wide[1, :, start : start + cols]
    w = torch.rand(cols + 1, device="cuda", generator=g)[1:]  # float32, off a 16-byte boundary
    w = w.clone() if start == 0 else w
    _check_norm(x, w, r, 1e-6, ops.rms_norm_fp8(x, w, r, return_normed=True))


def test_norm_keeps_leading_dimensions_and_a_bad_row_to_itself():
    g = _gen(2)
    x = torch.randn(2, 3, 4, 256, device="cuda", generator=g)
    w = torch.ones(256, device="cuda")
    q, s, h = ops.rms_norm_fp8(x, w)
    assert q.shape == x.shape and s.shape == (2, 3, 4, 2) and h is x
    bad = x.clone()
    bad[1, 0, 2, 5], bad[0, 1, 0, 6] = float("nan"), float("inf")
    q2, s2, _ = ops.rms_norm_fp8(bad, w)
    touched = torch.zeros(2, 3, 4, dtype=torch.bool, device="cuda")
    touched[1, 0, 2] = touched[0, 1, 0] = True
    assert torch.equal(_bits(q2)[~touched], _bits(q)[~touched]) and torch.equal(_bits(s2)[~touched], _bits(s)[~touched])
    assert q2[1, 0, 2].float().isnan().all()  # a row with NaN has no root mean square
    assert q2[0, 1, 0, 6].float().isnan() and (q2[0, 1, 0, :6].float() == 0).all()  # inf * 0, and the others over infinity


def test_norm_of_zeros_and_of_no_rows():
    x = torch.zeros(3, 200, device="cuda")
    q, s, _ = ops.rms_norm_fp8(x, torch.ones(200, device="cuda"), eps=0.0 + 1e-6)
    assert (q.float() == 0).all() and (_bits(s) == 1).all()
    q, s, h = ops.rms_norm_fp8(x[:0], torch.ones(200, device="cuda"), x[:0])
    assert q.shape == (0, 200) and s.shape == (0, 2) and h.shape == (0, 200)


# ------------------------------------------------------------------------------------------- products
def _operands(m, n, k, groups=None, seed=0):
    g = _gen(seed)
    a = torch.randn(m, k, device="cuda", generator=g) * torch.exp(torch.randn(1, k, device="cuda", generator=g))
    shape = (n, k) if groups is None else (groups, n, k)
    b = torch.randn(shape, device="cuda", generator=g) * torch.exp(torch.randn(*shape[:-1], 1, device="cuda", generator=g))
    return *ops.quantize_fp8(a), *ops.quantize_weight_fp8(b)


def _check_product(y, a, sa, b, sb, dtype):
    av, bv = reference.dequantize_fp8(a, sa, D), reference.dequantize_weight_fp8(b, sb, D)
    want, size = av @ bv.T, av.abs() @ bv.abs().T
    off = size * _sum_bound(a.shape[1], 32) + want.abs() * HALF[dtype]
    assert y.dtype == dtype and ((y.double() - want).abs() <= off).all()
    return want


PRODUCTS = [
    (1, 1, 16), (1, 128, 128), (16, 129, 112), (17, 127, 144), (1, 7168, 2048), (64, 4096, 7168), (37, 1000, 1040), (128, 300, 640), (129, 513, 2064),
    (256, 256, 1024), (257, 256, 128), (300, 520, 144), (1001, 700, 2064), (2000, 1111, 512), (8200, 64, 256),
]


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_product(m, n, k, out_dtype):
    a, sa, b, sb = _operands(m, n, k, seed=m)
    y = ops.matmul_fp8(a, sa, b, sb, out_dtype=out_dtype)
    _check_product(y, a, sa, b, sb, out_dtype)
    assert torch.equal(y, ops.matmul_fp8(a, sa, b, sb, out_dtype=out_dtype))  # the same bits every time
    assert ops.check() == 0


# rows in parts for the CTAs: parts that end inside a tile, one column, both sides of the step to CTA pairs
PRODUCTS_IN_PARTS = [
    (17, 9, 272), (176, 105, 528), (200, 1000, 1024), (257, 1, 16), (294, 117, 1232), (349, 863, 272), (772, 2164, 816), (1000, 2048, 1024),
    (1001, 1, 4096), (3916, 353, 1040), (3916, 353, 5568), (20011, 128, 144), (40001, 64, 272), (2304, 2048, 1536), (2305, 2049, 1536),
]


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n,k", PRODUCTS_IN_PARTS)
def test_product_of_rows_in_parts(m, n, k, out_dtype):
    a, sa, b, sb = _operands(m, n, k, seed=m + n)
    whole = torch.full((m + 3, n + 5), 3.0, device="cuda", dtype=out_dtype)
    y = ops.matmul_fp8(a, sa, b, sb, out=whole[:m, :n], out_dtype=out_dtype)
    _check_product(y, a, sa, b, sb, out_dtype)
    assert (whole[m:] == 3).all() and (whole[:, n:] == 3).all()
    assert torch.equal(y, ops.matmul_fp8(a, sa, b, sb, out_dtype=out_dtype))
    assert ops.check() == 0


@pytest.mark.parametrize("m", [5, 300])
def test_product_of_rows_apart_into_rows_apart(m):
    a, sa, b, sb = _operands(m, 200, 272)
    wide_a = torch.zeros(m, 320, device="cuda").to(torch.float8_e4m3fn)
    wide_a[:, 16:288].copy_(a)
    wide_s = torch.zeros(m, 7, dtype=torch.uint8, device="cuda")
    wide_s[:, 2:5] = _bits(sa)
    for ld, first in ((200, 0), (208, 0), (203, 1)):
        whole = torch.full((m, ld), 3.0, device="cuda", dtype=torch.bfloat16)
        out = whole[:, first : first + 200]
        y = ops.matmul_fp8(wide_a[:, 16:288], wide_s.view(torch.float8_e8m0fnu)[:, 2:5], b, sb, out=out)
        assert y.data_ptr() == out.data_ptr()
        _check_product(y, a, sa, b, sb, torch.bfloat16)
        assert (whole[:, :first] == 3).all() and (whole[:, first + 200 :] == 3).all()


@pytest.mark.parametrize("m", [3, 400])
def test_a_bad_row_or_scale_stays_with_itself(m):
    a, sa, b, sb = _operands(m, 384, 256)
    y = ops.matmul_fp8(a, sa, b, sb)
    a2, sa2, b2 = a.clone(), sa.clone(), b.clone()
    _bits(a2)[1, 7] = 0x7F  # NaN
    _bits(sa2)[2, 1] = 0xFF  # the scale that is NaN
    _bits(b2)[130, 0] = 0x7F
    z = ops.matmul_fp8(a2, sa2, b2, sb)
    keep = torch.ones_like(y, dtype=torch.bool)
    keep[1] = keep[2] = False
    keep[:, 130] = False
    assert torch.equal(z[keep], y[keep]) and z[~keep].isnan().all()


@pytest.mark.parametrize("m", [4, 300])
def test_scales_over_their_whole_range(m):
    a, sa, b, sb = _operands(m, 256, 512)
    down = torch.tensor([-60, -20, 20, 60], dtype=torch.int16, device="cuda")
    sa2 = (_bits(sa).to(torch.int16) + down).clamp(0, 254).to(torch.uint8).view(torch.float8_e8m0fnu)
    sb2 = (_bits(sb).to(torch.int16) - down).clamp(0, 254).to(torch.uint8).view(torch.float8_e8m0fnu)
    y = ops.matmul_fp8(a, sa2, b, sb2, out_dtype=torch.float32)
    _check_product(y, a, sa2, b, sb2, torch.float32)


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize(
    "rows,n,k,extra",
    [([3, 0, 5], 256, 128, 0), ([1], 100, 256, 4), ([0, 0], 64, 128, 3), ([300, 0, 1, 224, 225, 7], 520, 1040, 13), ([7] * 128, 40, 16, 0),
     ([33, 500, 2], 264, 656, 1)],
)
def test_groups(rows, n, k, extra, out_dtype):
    m = sum(rows) + extra
    a, sa, b, sb = _operands(m, n, k, len(rows))
    out = torch.full((m, n), 5.0, device="cuda", dtype=out_dtype)
    y = ops.matmul_fp8(a, sa, b, sb, rows=torch.tensor(rows, dtype=torch.int32, device="cuda"), out=out, out_dtype=out_dtype)
    at = 0
    for e, count in enumerate(rows):
        if count:
            _check_product(y[at : at + count], a[at : at + count], sa[at : at + count], b[e], sb[e], out_dtype)
        at += count
    assert (out[at:] == 5).all() and ops.check() == 0


def test_groups_with_counts_that_are_wrong():
    a, sa, b, sb = _operands(40, 256, 256, 3)
    rows = torch.tensor([-3, 30, 1000], dtype=torch.int32, device="cuda")  # none, 30, and no more than there are
    y = ops.matmul_fp8(a, sa, b, sb, rows=rows, out_dtype=torch.float32)
    _check_product(y[:30], a[:30], sa[:30], b[1], sb[1], torch.float32)
    _check_product(y[30:], a[30:], sa[30:], b[2], sb[2], torch.float32)


def test_no_rows():
    a, sa, b, sb = _operands(4, 64, 128)
    assert ops.matmul_fp8(a[:0], sa[:0], b, sb).shape == (0, 64)


# ------------------------------------------------------------------------------------------- the layer for a few tokens
def _layer(tokens, topk, experts, hidden, inter, fp8, seed=0):
    g = _gen(seed)
    x = torch.randn(tokens, hidden, device="cuda", generator=g).bfloat16()
    w13 = (torch.randn(experts, 2 * inter, hidden, device="cuda", generator=g) * hidden**-0.5).bfloat16()
    w2 = (torch.randn(experts, hidden, inter, device="cuda", generator=g) * inter**-0.5).bfloat16()
    gate, idx = torch.softmax(torch.randn(tokens, experts, device="cuda", generator=g), -1).topk(topk, -1)
    scales = {}
    if fp8:
        (w13, scales["w13_scale"]), (w2, scales["w2_scale"]) = ops.quantize_weight_fp8(w13), ops.quantize_weight_fp8(w2)
    return x, idx, gate, w13, w2, scales


def _oracle(x, idx, gate, w13, w2, scales, x_scale=None):
    """(result, bound) in 64 bits.  The bound: the roundings of both products' sums, the result's own, and one step for
    every activation that lies nearer to a rounding border than its own error."""
    fp8 = bool(scales)
    if fp8:
        xv = reference.dequantize_fp8(*(reference.quantize_fp8_reference(x) if x_scale is None else (x, x_scale)), D)
    else:
        xv = x.double()
    tokens, hidden = x.shape
    out, off = torch.zeros(tokens, hidden, dtype=D, device="cuda"), torch.zeros(tokens, hidden, dtype=D, device="cuda")
    per = 32 if fp8 else 16
    for e in idx[(idx >= 0) & (idx < w13.shape[0])].unique().tolist():
        tok, k = (idx == e).nonzero(as_tuple=True)
        up_gate = reference.dequantize_weight_fp8(w13[e], scales["w13_scale"][e], D) if fp8 else w13[e].double()
        down = reference.dequantize_weight_fp8(w2[e], scales["w2_scale"][e], D) if fp8 else w2[e].double()
        split = lambda v: (v.unflatten(-1, (-1, 2, 128))[:, :, i].flatten(1) for i in (0, 1))  # noqa: E731
        gt, up = split(xv[tok] @ up_gate.T)
        gt_off, up_off = (v * _sum_bound(hidden, per) for v in split(xv[tok].abs() @ up_gate.abs().T))
        act = gt * torch.sigmoid(gt) * up
        # silu's slope is at most 1.1; its exponential and quotient are good to 2**-20
        act_off = 1.1 * gt_off * up.abs() + (gt * torch.sigmoid(gt)).abs() * up_off + act.abs() * 2.0**-20
        if fp8:
            q, s = reference.quantize_fp8_reference(act)
            held = reference.dequantize_fp8(q, s, D)
            scale = reference.dequantize_fp8(torch.ones_like(q.float()).to(q.dtype), s, D)
            digit = (torch.frexp(act / scale)[1] - 1).clamp_min(-6)
            step = torch.exp2(digit.double() - 3) * scale
            top = act.abs().unflatten(-1, (-1, 128)).amax(-1) / (448 * scale[:, ::128])
            border = ((top.log2() - top.log2().round()).abs() < 2.0**-16).repeat_interleave(128, -1)  # the scale itself may go either way
        else:
            held = act.bfloat16().double()
            step = torch.exp2((torch.frexp(act)[1] - 1).double() - 7)
            border = torch.zeros_like(act, dtype=torch.bool)
        near = ((act - held).abs() + act_off >= step / 2) | border
        held_off = torch.where(near, 2 * step, torch.zeros_like(step))
        w = gate[tok, k].double().unsqueeze(1)
        out.index_add_(0, tok, held @ down.T * w)
        off.index_add_(0, tok, (held_off @ down.abs().T + held.abs() @ down.abs().T * (_sum_bound(w2.shape[2], per) + 2.0**-20)) * w.abs())
    return out, off + out.abs() * 2.0**-8


def _check_layer(y, *args, **kw):
    want, off = _oracle(*args, **kw)
    assert ((y.double() - want).abs() <= off).all()
    # most results are far nearer: the bound above lets a step through only where a border is near
    assert float((y.double() - want).norm()) <= 2.0**-7 * float(want.norm())


LAYERS = [
    (1, 1, 1, 256, 128), (1, 8, 16, 7168, 2048), (2, 1, 300, 256, 128), (5, 2, 8, 512, 256), (12, 4, 32, 1024, 512), (16, 4, 16, 768, 384),
    (17, 4, 16, 1280, 640), (33, 8, 32, 1024, 512), (64, 8, 48, 2048, 1024), (64, 32, 64, 256, 128), (40, 1, 2, 768, 640), (3, 2, 512, 256, 128),
    (7, 3, 5, 2304, 1152), (64, 1, 1, 512, 256),
]


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("tokens,topk,experts,hidden,inter", LAYERS)
def test_few_tokens(tokens, topk, experts, hidden, inter, fp8):
    x, idx, gate, w13, w2, scales = _layer(tokens, topk, experts, hidden, inter, fp8, seed=tokens)
    y = ops.moe_few_tokens(x, idx, gate, w13, w2, **scales)
    _check_layer(y, x, idx, gate, w13, w2, scales)
    for _ in range(3):
        assert torch.equal(y, ops.moe_few_tokens(x, idx, gate, w13, w2, **scales))
    if fp8:
        q, s = ops.quantize_fp8(x)
        assert torch.equal(y, ops.moe_few_tokens(q, idx, gate, w13, w2, x_scale=s, **scales))
    assert ops.check() == 0


@pytest.mark.parametrize("fp8", [False, True])
def test_few_tokens_of_choices_that_are_empty_wrong_or_made_twice(fp8):
    x, idx, gate, w13, w2, scales = _layer(6, 3, 8, 512, 256, fp8)
    idx = torch.tensor([[-1, -1, -1], [2, 2, 2], [8, 1, -7], [5, -1, 5], [0, 1, 2], [1 << 40, 3, -(1 << 40)]], device="cuda")
    y = ops.moe_few_tokens(x, idx, gate, w13, w2, **scales)
    _check_layer(y, x, idx, gate, w13, w2, scales)
    assert (y[0] == 0).all()
    none = ops.moe_few_tokens(x, torch.full_like(idx, -1), gate, w13, w2, **scales)
    assert none.shape == y.shape and (none == 0).all()
    assert ops.moe_few_tokens(x[:0], idx[:0], gate[:0], w13, w2, **scales).shape == (0, 512)


def test_few_tokens_types_and_strides():
    x, idx, gate, w13, w2, scales = _layer(9, 2, 8, 512, 256, True)
    y = ops.moe_few_tokens(x, idx, gate, w13, w2, **scales)
    wide = torch.zeros(9, 640, device="cuda", dtype=torch.bfloat16)
    wide[:, 64:576] = x
    assert torch.equal(y, ops.moe_few_tokens(wide[:, 64:576], idx.int(), gate, w13, w2, **scales))
    assert torch.equal(y, ops.moe_few_tokens(x, idx.t().contiguous().t(), gate.t().contiguous().t(), w13, w2, **scales))
    half = gate.bfloat16()
    z = ops.moe_few_tokens(x, idx, half, w13, w2, **scales)
    assert torch.equal(z, ops.moe_few_tokens(x, idx, half.float(), w13, w2, **scales))
    q, s = ops.quantize_fp8(x)
    wide_s = torch.zeros(9, 9, dtype=torch.uint8, device="cuda")
    wide_s[:, 3:7] = _bits(s)
    assert torch.equal(y, ops.moe_few_tokens(q, idx, gate, w13, w2, x_scale=wide_s.view(torch.float8_e8m0fnu)[:, 3:7], **scales))


@pytest.mark.parametrize("fp8", [False, True])
def test_few_tokens_keep_a_bad_token_and_a_bad_expert_to_themselves(fp8):
    x, idx, gate, w13, w2, scales = _layer(8, 2, 6, 512, 256, fp8)
    idx = torch.tensor([[0, 1], [1, 2], [2, 3], [3, 4], [0, 2], [4, 1], [2, 4], [5, 5]], device="cuda")
    y = ops.moe_few_tokens(x, idx, gate, w13, w2, **scales)
    bad = x.clone()
    bad[4, 3] = float("nan")
    w13_bad = w13.clone()
    if fp8:
        _bits(w13_bad)[5, 0, 0] = 0x7F
    else:
        w13_bad[5, 0, 0] = float("inf")
    z = ops.moe_few_tokens(bad, idx, gate, w13_bad, w2, **scales)
    keep = torch.ones(8, dtype=torch.bool, device="cuda")
    keep[4] = keep[7] = False
    assert torch.equal(z[keep], y[keep])
    assert not z[4].isfinite().any() and not z[7].isfinite().all()


def test_everything_in_one_captured_graph_replayed_on_new_inputs():
    """norm -> layer for a few tokens, and a product of the same rows, as a decode step runs them."""
    tokens, hidden = 6, 512
    x, idx, gate, w13, w2, scales = _layer(tokens, 2, 8, hidden, 256, True)
    wq, ws = ops.quantize_weight_fp8(torch.randn(384, hidden, device="cuda", generator=_gen(9)))
    weight = torch.rand(hidden, device="cuda", generator=_gen(8)).bfloat16() + 0.5
    r = torch.zeros_like(x)

    def step():
        q, s, h = ops.rms_norm_fp8(x, weight, r)
        return ops.moe_few_tokens(q, idx, gate, w13, w2, x_scale=s, **scales), ops.matmul_fp8(q, s, wq, ws), h

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
        graphs = []
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                out = step()
            graphs.append((graph, out))
    torch.cuda.synchronize()
    for i in range(4):
        g = _gen(20 + i)
        x.copy_(torch.randn(tokens, hidden, device="cuda", generator=g))
        r.copy_(torch.randn(tokens, hidden, device="cuda", generator=g))
        idx.copy_(torch.randint(-1, 8, idx.shape, device="cuda", generator=g))
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        graphs[0][0].replay()  # both graphs at once, on two streams
        with torch.cuda.stream(side):
            graphs[1][0].replay()
        torch.cuda.synchronize()
        want = step()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))
    assert ops.check() == 0


def test_calls_at_once_on_several_streams_share_nothing():
    cases = [_layer(t, 4, 16, 1024, 512, fp8, seed=t) for t, fp8 in ((3, True), (30, False), (64, True), (11, False))]
    want = [ops.moe_few_tokens(*c[:5], **c[5]) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[] for _ in cases]
    for _ in range(6):
        for i, (c, stream) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(stream):
                got[i].append(ops.moe_few_tokens(*c[:5], **c[5]))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i, ys in enumerate(got) for y in ys) and ops.check() == 0


def test_passes_follow_one_another_without_a_gap():
    """Kernels start while their predecessors run out, the buffers of the pass before them still in use."""
    batches = [_layer(t, 4, 16, 1024, 512, True, seed=t) for t in (1, 20, 64)]
    weight = torch.ones(1024, device="cuda", dtype=torch.bfloat16)

    def step(b):
        x, idx, gate, w13, w2, scales = b
        q, s, _ = ops.rms_norm_fp8(x, weight, x)
        y = ops.moe_few_tokens(q, idx, gate, w13, w2, x_scale=s, **scales)
        q, s = ops.quantize_fp8(y)
        return ops.matmul_fp8(q, s, w2[0].view(torch.uint8).view(1024, 512)[:, :].reshape(512, 1024).view(torch.float8_e4m3fn), _scale_ones(4, 8))

    def _scale_ones(n, k):
        return torch.full((n, k), 127, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)

    want = []
    for b in batches:
        want.append(step(b))
        torch.cuda.synchronize()
    got = [step(b) for _ in range(8) for b in batches]
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i % 3]) for i, y in enumerate(got))


# ------------------------------------------------------------------------------------------- refusals on the device
def test_arguments_that_are_refused():
    a, sa, b, sb = _operands(4, 64, 128)
    x, idx, gate, w13, w2, scales = _layer(3, 2, 4, 256, 128, True)
    refused = [
        (lambda: ops.matmul_fp8(a[:, 8:120], sa, b[:, 8:120].contiguous(), sb), "16-byte"),
        (lambda: ops.matmul_fp8(a, sa.cpu(), b, sb), "a_scale"),
        (lambda: ops.matmul_fp8(a, sa, b.t().contiguous().t(), sb), "contiguous"),
        (lambda: ops.matmul_fp8(a, sa, b, sb, out=torch.empty(4, 64, device="cuda")), "out must"),
        (lambda: ops.matmul_fp8(a, sa, b, sb, rows=torch.ones(1, dtype=torch.int32, device="cuda")), "b must"),
        (lambda: ops.matmul_fp8(a, sa, b[None], sb[None], rows=torch.ones(1, dtype=torch.int64, device="cuda")), "rows must"),
        (lambda: ops.quantize_fp8(torch.zeros(2, 20000, device="cuda")), "1 to 16384"),
        (lambda: ops.quantize_fp8(torch.zeros(4, 8, device="cuda").t()), "next to one another"),
        (lambda: ops.quantize_fp8(torch.zeros(4, 8, device="cuda", requires_grad=True)), "gradient"),
        (lambda: ops.rms_norm_fp8(x, torch.ones(256, device="cuda").half()), "float32 or of x's type"),
        (lambda: ops.rms_norm_fp8(x, torch.ones(256)), "on x's device"),
        (lambda: ops.moe_few_tokens(x.repeat(30, 1), idx.repeat(30, 1), gate.repeat(30, 1), w13, w2, **scales), "at most 64"),
        (lambda: ops.moe_few_tokens(x, idx.float(), gate, w13, w2, **scales), "idx must"),
        (lambda: ops.moe_few_tokens(x, idx, gate, w13, w2, w13_scale=scales["w13_scale"]), "come together"),
        (lambda: ops.moe_few_tokens(x.half(), idx, gate, w13, w2, **scales), "x must be"),
        (lambda: ops.moe_few_tokens(x, idx, gate, w13, w2, w13_scale=scales["w2_scale"], w2_scale=scales["w13_scale"]), "scales of"),
        (lambda: ops.moe_few_tokens(x[:, :128], idx, gate, w13, w2, **scales), "multiple of 256"),
    ]
    for call, words in refused:
        with pytest.raises(ValueError, match=words):
            call()
    with torch.no_grad():
        ops.quantize_fp8(torch.zeros(4, 8, device="cuda", requires_grad=True))
    torch.cuda.synchronize()


# ------------------------------------------------------------------------------------------- far offsets, many launches at once
def test_rows_behind_two_to_the_31_values():
    rows, cols = 270_000, 8192
    x = torch.zeros(rows, cols, device="cuda", dtype=torch.bfloat16)
    last = torch.randn(3, cols, device="cuda", generator=_gen(4)).bfloat16()
    x[-3:] = last
    w = torch.ones(cols, device="cuda", dtype=torch.bfloat16)
    got = ops.rms_norm_fp8(x, w, x)
    want = ops.rms_norm_fp8(last, w, last)
    for a, b in zip(got, want):
        assert torch.equal(a[-3:].view(torch.uint8), b.view(torch.uint8))
    assert not got[0][0].float().any() and (_bits(got[1])[0] == 1).all()  # a block of zeros has the smallest scale


def test_results_behind_two_to_the_31_values():
    m, n, k = 70_000, 32_768, 32
    a, sa, b, sb = _operands(64, n, k)
    many, many_s = torch.zeros(m, k, device="cuda").to(torch.float8_e4m3fn), torch.full((m, 1), 127, dtype=torch.uint8, device="cuda")
    many[-64:].copy_(a)
    many_s[-64:] = _bits(sa)
    y = ops.matmul_fp8(many, many_s.view(torch.float8_e8m0fnu), b, sb)
    _check_product(y[-64:], a, sa, b, sb, torch.bfloat16)
    assert not y[:64].any()


def test_weights_behind_two_to_the_31_bytes():
    x, idx, gate, w13, w2, scales = _layer(5, 2, 2, 2048, 2048, True)
    experts = 300
    far = {n: torch.zeros(experts, *t.shape[1:], dtype=torch.uint8, device="cuda") for n, t in (("w13", w13), ("w2", w2), *scales.items())}
    for n, t in (("w13", w13), ("w2", w2), *scales.items()):
        far[n][-2:] = _bits(t)
    typed = {n: t.view(torch.float8_e8m0fnu if "scale" in n else torch.float8_e4m3fn) for n, t in far.items()}
    y = ops.moe_few_tokens(x, idx, gate, w13, w2, **scales)
    assert torch.equal(y, ops.moe_few_tokens(x, idx + experts - 2, gate, **typed))


def test_products_of_many_sizes_at_once_on_several_streams():
    """Clusters of several launches share SMs; none may wait for another's tensor memory."""
    cases = [_operands(m, n, k, seed=m) for m, n, k in ((1, 7168, 2048), (33, 300, 256), (48, 4096, 128), (100, 512, 2064), (200, 1000, 512), (250, 256, 7168))]
    want = [ops.matmul_fp8(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[] for _ in cases]
    for i in range(20):
        for j in range(len(cases)):
            c = (i + j) % len(cases)
            with torch.cuda.stream(streams[j]):
                got[c].append(ops.matmul_fp8(*cases[c]))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i, ys in enumerate(got) for y in ys) and ops.check() == 0

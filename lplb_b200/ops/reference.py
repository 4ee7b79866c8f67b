"""Plain PyTorch restatements of the planner kernels.

They run on any device, define the semantics the CUDA kernels are tested against, and
are what ``Planner`` executes when it is built on a CPU device.

* ``count_reference``   – histogram with a per-slice inclusive prefix
  (kernel: ``count_kernel`` in ``csrc/planner_kernels.cuh``).
* ``quotas_reference``  – integer number of each expert's local tokens that stay on the
  original, ``rint(share * total)``.
* ``redirect_reference`` – logical -> physical rewrite with the even-spread rule
  (kernel: ``redirect_kernel``).  Tokens of one expert are numbered in array order here;
  the kernels number them in an order that depends on atomics, so outputs agree as
  multisets per expert, not position by position.

The 8-bit serving operators (``lplb_b200.ops.fp8``) are restated below in 32 bits, or in 64 where their
inputs are: ``quantize_fp8_reference``, ``rms_norm_fp8_reference``, ``matmul_fp8_reference``,
``moe_few_tokens_reference``.  So are the operators around a layer's experts (``lplb_b200.ops.experts``):
``gate_topk_reference``, ``expert_order_reference``, ``take_rows_reference``, ``combine_rows_reference`` and the
gradients of the first and the last, and the product with an epilogue (``lplb_b200.ops.dense``) with its gradients,
``matmul_reference`` and ``matmul_backward_reference``.
"""

from __future__ import annotations

import torch

__all__ = [
    "slice_bounds",
    "count_reference",
    "quotas_reference",
    "redirect_reference",
    "dequantize_fp8",
    "dequantize_weight_fp8",
    "quantize_fp8_reference",
    "quantize_weight_fp8_reference",
    "rms_norm_fp8_reference",
    "matmul_fp8_reference",
    "moe_few_tokens_reference",
    "gate_topk_reference",
    "gate_topk_backward_reference",
    "expert_order_reference",
    "take_rows_reference",
    "combine_rows_reference",
    "combine_rows_backward_reference",
    "matmul_reference",
    "matmul_backward_reference",
]

_BLOCK = 256


def slice_bounds(n: int, n_slices: int, align: int = _BLOCK) -> list[int]:
    """Token range boundaries of the kernels' CTA slices (``slice_begin`` in ``common.cuh``)."""
    per = -(-n // n_slices)
    per = -(-per // align) * align
    return [min(n, per * p) for p in range(n_slices + 1)]


def count_reference(idx: torch.Tensor, n_logical: int, n_slices: int) -> tuple[torch.Tensor, torch.Tensor]:
    """``(counts [E], inclusive prefix over slices [n_slices, E])``, int32; ``-1`` is skipped."""
    flat = idx.reshape(-1).long()
    bounds = slice_bounds(flat.numel(), n_slices)
    rows = torch.zeros(n_slices, n_logical + 1, dtype=torch.int64, device=idx.device)
    for p in range(n_slices):
        part = flat[bounds[p] : bounds[p + 1]]
        valid = (part >= 0) & (part < n_logical)
        part = torch.where(valid, part, torch.full_like(part, n_logical))
        rows[p].scatter_add_(0, part, torch.ones_like(part))
    prefix = rows[:, :n_logical].cumsum(0).to(torch.int32)
    return prefix[-1].clone(), prefix


def quotas_reference(total: torch.Tensor, probs: torch.Tensor, log2edge: torch.Tensor) -> torch.Tensor:
    """Tokens of each expert kept on the original: all of them for unreplicated experts."""
    p = probs.reshape(-1).float()
    p = torch.where(torch.isnan(p), torch.full_like(p, 0.5), p).clamp(0, 1)
    edge = log2edge.long()
    share = torch.where(edge >= 0, p[edge.clamp_min(0)], torch.ones_like(total, dtype=torch.float32))
    q = torch.round(share * total.float()).to(torch.int64)  # round-half-even, like cvt.rni
    return torch.minimum(q.clamp_min(0), total.long())


def redirect_reference(
    idx: torch.Tensor, probs: torch.Tensor, log2phy: torch.Tensor, log2edge: torch.Tensor
) -> torch.Tensor:
    """Rewrite logical ids to physical ids; ``-1`` (and out-of-range ids) map to ``-1``."""
    n_logical = log2phy.shape[0]
    flat = idx.reshape(-1).long()
    valid = (flat >= 0) & (flat < n_logical)
    safe = torch.where(valid, flat, torch.zeros_like(flat))
    total = torch.zeros(n_logical, dtype=torch.int64, device=idx.device)
    total.scatter_add_(0, safe, valid.long())
    quota = quotas_reference(total, probs.to(idx.device), log2edge.to(idx.device))
    # ordinal of every token among the tokens of its expert, in array order
    order = torch.sort(torch.where(valid, flat, torch.full_like(flat, n_logical)), stable=True)
    starts = torch.zeros(n_logical + 2, dtype=torch.int64, device=idx.device)
    starts[1 : n_logical + 1] = total.cumsum(0)
    ordinal = torch.empty_like(flat)
    ordinal[order.indices] = torch.arange(flat.numel(), device=idx.device) - starts[order.values.clamp_max(n_logical)]
    tot = total[safe].clamp_min(1)
    quo = quota[safe]
    keep = (quo >= tot) | ((quo > 0) & ((ordinal * quo) % tot + quo >= tot))
    phys = log2phy.to(idx.device).long()
    keep = keep | (phys[safe, 1] < 0)
    out = torch.where(keep, phys[safe, 0], phys[safe, 1])
    out = torch.where(valid, out, torch.full_like(out, -1))
    return out.reshape(idx.shape).to(idx.dtype)


# ---------------------------------------------------------------------------- values in 8 bits
_SCALE_BLOCK = 128


def _wide(x: torch.Tensor) -> torch.Tensor:
    return x if x.dtype == torch.float64 else x.float()


def _scale_exponents(amax: torch.Tensor) -> torch.Tensor:
    """Biased exponent of the smallest power of two ``s`` with ``amax / s <= 448`` (``scale_exponent`` in
    ``fp8.cuh``): 448 is 1.75 * 2**8, so it is amax's exponent less 8, one more above a mantissa of 1.75."""
    mantissa, exponent = torch.frexp(amax)  # mantissa in [0.5, 1)
    e = exponent - 1 - 8 + (mantissa > 0.875).to(exponent.dtype) + 127
    return torch.where(amax > 0, e, torch.ones_like(e)).clamp_min(1).to(torch.uint8)


def _powers(scale: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    byte = scale.view(torch.uint8)
    power = torch.ldexp(torch.ones((), dtype=dtype, device=scale.device), byte.to(dtype) - 127)
    return torch.where(byte == 255, torch.full_like(power, float("nan")), power)  # the one byte of the type that is no power


def dequantize_fp8(q: torch.Tensor, scale: torch.Tensor, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values that rows in 8 bits stand for."""
    return q.to(dtype) * _powers(scale, dtype).repeat_interleave(_SCALE_BLOCK, -1)[..., : q.shape[-1]]


def dequantize_weight_fp8(q: torch.Tensor, scale: torch.Tensor, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values that weights in 8 bits stand for."""
    s = _powers(scale, dtype).repeat_interleave(_SCALE_BLOCK, -1)[..., : q.shape[-1]]
    return q.to(dtype) * s.repeat_interleave(_SCALE_BLOCK, -2)[..., : q.shape[-2], :]


def _to_e4m3(x: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    x = torch.where(x.isfinite(), x, torch.full_like(x, float("nan")))
    return (x / _powers(scale, x.dtype)).to(torch.float8_e4m3fn)


def quantize_fp8_reference(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows to e4m3 with a scale per 128 (kernel: ``row_fp8_kernel`` in ``csrc/norm_fp8.cu``)."""
    f = _wide(x)
    k = f.shape[-1]
    blocks = torch.nn.functional.pad(f, (0, -k % _SCALE_BLOCK)).unflatten(-1, (-1, _SCALE_BLOCK))
    magnitude = torch.where(blocks.isfinite(), blocks.abs(), torch.zeros_like(blocks))
    e = _scale_exponents(magnitude.amax(-1))
    return _to_e4m3(blocks, e.unsqueeze(-1)).flatten(-2)[..., :k].contiguous(), e.view(torch.float8_e8m0fnu)


def quantize_weight_fp8_reference(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Weights to e4m3 with a scale per 128 x 128 (kernel: ``weight_fp8_kernel``)."""
    f = _wide(w)
    n, k = f.shape[-2:]
    padded = torch.nn.functional.pad(f, (0, -k % _SCALE_BLOCK, 0, -n % _SCALE_BLOCK))
    blocks = padded.unflatten(-1, (-1, _SCALE_BLOCK)).unflatten(-3, (-1, _SCALE_BLOCK))
    magnitude = torch.where(blocks.isfinite(), blocks.abs(), torch.zeros_like(blocks))
    e = _scale_exponents(magnitude.amax((-3, -1)))
    q = _to_e4m3(blocks, e.unsqueeze(-1).unsqueeze(-3)).flatten(-2).flatten(-3, -2)
    return q[..., :n, :k].contiguous(), e.view(torch.float8_e8m0fnu)


def rms_norm_fp8_reference(
    x: torch.Tensor,
    weight: torch.Tensor,
    residual: torch.Tensor | None = None,
    eps: float = 1e-6,
    return_normed: bool = False,
) -> tuple[torch.Tensor, ...]:
    """Residual's addition, norm and conversion to 8 bits; the sum is rounded to ``x``'s type before its norm is taken."""
    h = x if residual is None else (_wide(x) + _wide(residual)).to(x.dtype)
    f = _wide(h)
    n = f * torch.rsqrt((f * f).mean(-1, keepdim=True) + eps) * weight.to(f.dtype)
    out = (*quantize_fp8_reference(n), h)
    return (*out, n.to(x.dtype)) if return_normed else out


def matmul_fp8_reference(
    a: torch.Tensor,
    a_scale: torch.Tensor,
    b: torch.Tensor,
    b_scale: torch.Tensor,
    rows: torch.Tensor | None = None,
    dtype: torch.dtype = torch.float32,
) -> torch.Tensor:
    """``a @ b.T`` of the values they stand for; with ``rows`` the groups of ``a``'s rows, one after the other, each
    with its own matrix of ``b`` (rows behind the last group are zero here)."""
    af, bf = dequantize_fp8(a, a_scale, dtype), dequantize_weight_fp8(b, b_scale, dtype)
    if rows is None:
        return af @ bf.T
    out = torch.zeros(a.shape[0], b.shape[1], dtype=dtype, device=a.device)
    at = 0
    for e, n in enumerate(rows.clamp_min(0).tolist()):
        out[at : at + n] = af[at : at + n] @ bf[e].T
        at += n
    return out


def moe_few_tokens_reference(
    x: torch.Tensor,
    idx: torch.Tensor,
    weights: torch.Tensor,
    w13: torch.Tensor,
    w2: torch.Tensor,
    x_scale: torch.Tensor | None = None,
    w13_scale: torch.Tensor | None = None,
    w2_scale: torch.Tensor | None = None,
    dtype: torch.dtype = torch.float32,
) -> torch.Tensor:
    """The layer of ``moe_few_tokens`` expert by expert, computed and returned in ``dtype``; activations are rounded as
    the kernels round them (bfloat16, or 8 bits where the weights are)."""
    fp8 = w13_scale is not None
    if fp8 and x_scale is None:
        x, x_scale = quantize_fp8_reference(x)
    xf = dequantize_fp8(x, x_scale, dtype) if fp8 else x.to(dtype)
    out = torch.zeros(x.shape[0], w2.shape[1], dtype=dtype, device=x.device)
    for e in idx[(idx >= 0) & (idx < w13.shape[0])].unique().tolist():
        tok, k = (idx == e).nonzero(as_tuple=True)
        up_gate = dequantize_weight_fp8(w13[e], w13_scale[e], dtype) if fp8 else w13[e].to(dtype)
        down = dequantize_weight_fp8(w2[e], w2_scale[e], dtype) if fp8 else w2[e].to(dtype)
        both = (xf[tok] @ up_gate.T).unflatten(-1, (-1, 2, _SCALE_BLOCK))
        gate, up = both[:, :, 0].flatten(1), both[:, :, 1].flatten(1)
        act = torch.nn.functional.silu(gate) * up
        act = dequantize_fp8(*quantize_fp8_reference(act), dtype) if fp8 else act.bfloat16().to(dtype)
        out.index_add_(0, tok, act @ down.T * weights[tok, k].to(dtype).unsqueeze(1))
    return out


def _scores(x: torch.Tensor, most: torch.Tensor, score: str, renormalize: bool) -> torch.Tensor:
    """Scores of logits ``x`` in rows whose largest is ``most`` (finite); for a renormalised weight up to a factor of the row."""
    if score == "softmax":
        return torch.exp(x - most)
    over = most.clamp_max(0) if renormalize else torch.zeros_like(most)
    return torch.exp(x.clamp_max(0) - over) / (1 + torch.exp(-x.abs()))


def gate_topk_reference(
    logits: torch.Tensor, topk: int, score: str = "softmax", renormalize: bool = False, scale: float = 1.0
) -> tuple[torch.Tensor, torch.Tensor]:
    """``(weights, idx)`` of the largest logits (kernel: ``gate_kernel`` in ``csrc/gate.cu``)."""
    x = _wide(logits)
    top, idx = torch.sort(x, dim=-1, descending=True, stable=True)  # NaN first; equal ones in the order of experts
    top, idx = top[:, :topk], idx[:, :topk]
    there = ~torch.isneginf(top)
    most = torch.where(there[:, :1], top[:, :1], torch.zeros_like(top[:, :1]))
    w = torch.where(there, _scores(top, most, score, renormalize), torch.zeros_like(top))
    if renormalize:
        w = w / torch.where(there[:, :1], w.sum(-1, keepdim=True), torch.ones_like(most))
    elif score == "softmax":
        w = w / torch.where(there[:, :1], _scores(x, most, score, False).sum(-1, keepdim=True), torch.ones_like(most))
    return torch.where(there, scale * w, torch.zeros_like(w)), torch.where(there, idx, torch.full_like(idx, -1))


def gate_topk_backward_reference(
    logits: torch.Tensor, idx: torch.Tensor, dweights: torch.Tensor, score: str = "softmax", renormalize: bool = False, scale: float = 1.0
) -> torch.Tensor:
    """The logits' gradient (kernel: ``gate_backward_kernel``)."""
    x = _wide(logits)
    there = idx >= 0
    at = idx.clamp_min(0)
    mine = torch.where(there, x.gather(1, at), torch.zeros_like(x[:, :1]))
    w = gate_topk_reference(logits, idx.shape[1], score, renormalize)[0]
    d = torch.where(there, scale * dweights.to(x.dtype), torch.zeros_like(w))
    along = (d * w).sum(-1, keepdim=True)
    dx = torch.zeros_like(x)
    if renormalize:
        each = w * (d - along)
    else:
        each = w * d
        if score == "softmax":
            alive = there[:, :1].expand_as(x)
            p = torch.softmax(torch.where(alive, x, torch.zeros_like(x)), -1)
            dx = torch.where(alive, -along * p, dx)
    if score == "sigmoid":
        each = each / (1 + torch.exp(mine))
    dx.scatter_add_(1, at, torch.where(there, each, torch.zeros_like(each)))
    return dx.to(logits.dtype)


def expert_order_reference(idx: torch.Tensor, n_experts: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(counts, place, source)`` of a stable sort by expert (kernel: ``order_kernel`` in ``csrc/expert_rows.cu``)."""
    flat = idx.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < n_experts), flat, torch.full_like(flat, n_experts))
    key, pair = torch.sort(key, stable=True)
    there = key < n_experts
    at = torch.arange(flat.numel(), device=flat.device)
    counts = torch.bincount(key, minlength=n_experts + 1)[:n_experts]
    place = torch.empty_like(flat)
    place[pair] = torch.where(there, at, torch.full_like(at, -1))
    return counts.int(), place.view(idx.shape).int(), torch.where(there, pair, torch.full_like(pair, -1)).int()


def take_rows_reference(x: torch.Tensor, place: torch.Tensor, source: torch.Tensor) -> torch.Tensor:
    """A row for every choice, in the order of experts; zeros behind the last (kernel: ``take_rows_kernel``)."""
    raw = x if x.element_size() > 1 else x.view(torch.uint8)
    if raw.shape[0] == 0:
        return x.new_empty(0, x.shape[1])
    rows = raw[source.clamp_min(0).long() // place.shape[1]]
    rows = torch.where((source >= 0).unsqueeze(1), rows, torch.zeros_like(rows))
    return rows if rows.dtype == x.dtype else rows.view(x.dtype)  # (a view by type has no forward-mode derivative)


def combine_rows_reference(rows: torch.Tensor, place: torch.Tensor, weights: torch.Tensor | None = None) -> torch.Tensor:
    """The rows of a token's choices, weighted and added up, rounded once (kernel: ``combine_rows_kernel``)."""
    out = _wide(rows.new_zeros(place.shape[0], rows.shape[1]))
    for k in range(place.shape[1] if rows.shape[0] else 0):
        there, at = (place[:, k] >= 0).unsqueeze(1), place[:, k].clamp_min(0).long()
        y = _wide(rows[at])
        out += torch.where(there, y if weights is None else y * weights[:, k : k + 1].to(y.dtype), torch.zeros_like(y))
    return out.to(rows.dtype)


def combine_rows_backward_reference(
    dout: torch.Tensor, rows: torch.Tensor, place: torch.Tensor, weights: torch.Tensor
) -> tuple[torch.Tensor, torch.Tensor]:
    """Gradients of rows and weights (kernel: ``combine_rows_backward_kernel``)."""
    d, y = _wide(dout), _wide(rows)
    drows, dweights = torch.zeros_like(y), d.new_zeros(place.shape)
    for k in range(place.shape[1] if rows.shape[0] else 0):
        token = (place[:, k] >= 0).nonzero().squeeze(1)
        at = place[token, k].long()
        drows[at] = d[token] * weights[token, k : k + 1].to(d.dtype)
        dweights[token, k] = (d[token] * y[at]).sum(-1)
    return drows.to(rows.dtype), dweights


def _groups(m: int, rows: torch.Tensor | None) -> list[tuple[int | None, slice]]:
    """``(matrix, rows of a)``; one matrix has no number."""
    if rows is None:
        return [(None, slice(0, m))]
    parts, at = [], 0
    for e, n in enumerate(rows.clamp_min(0).tolist()):
        parts.append((e, slice(at, min(m, at + n))))
        at = min(m, at + n)
    return parts


def _normal_cdf(z: torch.Tensor) -> torch.Tensor:
    return 0.5 * torch.special.erfc(-z * 0.5**0.5)


def _activated(z: torch.Tensor, activation: str | None) -> torch.Tensor:
    if activation == "relu":
        return z.clamp_min(0)
    if activation == "gelu":
        return z * _normal_cdf(z)
    if activation == "silu":
        return z * torch.sigmoid(z)
    if activation == "swiglu":
        gate, up = z.unflatten(-1, (-1, 2, _SCALE_BLOCK)).unbind(-2)
        return (gate * torch.sigmoid(gate) * up).flatten(-2)
    return z


def _through_activation(dout: torch.Tensor, z: torch.Tensor, activation: str) -> torch.Tensor:
    if activation == "relu":
        return torch.where(z > 0, dout, torch.zeros_like(dout))
    if activation == "gelu":
        return dout * (_normal_cdf(z) + z * torch.exp(-0.5 * z * z) * (2 * torch.pi) ** -0.5)
    if activation == "silu":
        s = torch.sigmoid(z)
        return dout * s * (1 + z * (1 - s))
    gate, up = z.unflatten(-1, (-1, 2, _SCALE_BLOCK)).unbind(-2)
    d, s = dout.unflatten(-1, (-1, _SCALE_BLOCK)), torch.sigmoid(gate)
    return torch.stack((d * up * s * (1 + gate * (1 - s)), d * gate * s), -2).flatten(-3)


def matmul_reference(
    a: torch.Tensor,
    b: torch.Tensor,
    bias: torch.Tensor | None = None,
    activation: str | None = None,
    residual: torch.Tensor | None = None,
    rows: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """``(act(z) + residual, z)`` with ``z = a @ b.T + bias`` (kernels: ``pair_matmul_kernel`` and ``few_product_kernel`` in
    ``csrc/matmul.cuh`` and ``matmul_few.cuh``); rows behind the last group have no product."""
    af = _wide(a)
    z = af.new_zeros(a.shape[0], b.shape[-2])
    out = af.new_zeros(a.shape[0], b.shape[-2] // (2 if activation == "swiglu" else 1))
    for e, part in _groups(a.shape[0], rows):
        here = af[part] @ _wide(b if e is None else b[e]).T
        if bias is not None:
            here = here + _wide(bias if e is None else bias[e]).to(here.dtype)
        z[part], out[part] = here, _activated(here, activation)
    return (out if residual is None else out + _wide(residual).to(out.dtype)), z


def _as_operand(dz: torch.Tensor, dtype: torch.dtype, dim: int) -> torch.Tensor:
    """``dz`` as a product's operand holds it.  In float16 it is held in parts of a power of two of its largest finite magnitude along ``dim``
    (``part_of`` in ``csrc/matmul.cuh``): its own numbers would end at 65504 and 2**-24."""
    if dtype != torch.float16 or dz.numel() == 0:
        return dz.to(dtype).to(dz.dtype)
    most = torch.where(dz.isfinite(), dz.abs(), torch.zeros_like(dz)).amax(dim, keepdim=True)
    exponent = torch.frexp(most).exponent.clamp_min(-111) - 15
    return torch.ldexp(torch.ldexp(dz, -exponent).to(dtype).to(dz.dtype), exponent)


def matmul_backward_reference(
    dout: torch.Tensor, a: torch.Tensor, b: torch.Tensor, z: torch.Tensor | None, activation: str | None = None, rows: torch.Tensor | None = None
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(da, db, dbias)``; ``z`` is what the activation was taken of."""
    af, bf = _wide(a), _wide(b)
    da, db, dbias = torch.zeros_like(af), torch.zeros_like(bf), bf.new_zeros(b.shape[:-1])
    for e, part in _groups(a.shape[0], rows):
        dz = _wide(dout[part]).to(af.dtype)
        if activation is not None:
            dz = _through_activation(dz, _wide(z[part]).to(af.dtype), activation)
        at = slice(None) if e is None else e
        dbias[at] = dz.sum(0)
        da[part], db[at] = _as_operand(dz, a.dtype, 1) @ bf[at], _as_operand(dz, a.dtype, 0).T @ af[part]
    return da, db, dbias

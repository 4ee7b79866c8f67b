"""Serving operators with values in 8 bits.

Values are ``torch.float8_e4m3fn``; every block of 128 along a row shares one power-of-two scale,
a ``torch.float8_e8m0fnu`` (weights: every block of 128 x 128).  That is the form whose scales the
B200's tensor cores multiply in by themselves.  A block's scale is the smallest power of two that
brings its largest finite magnitude to 448 or below, 2**-126 at least; infinities and NaN become NaN.

* :func:`quantize_fp8`, :func:`quantize_weight_fp8` – to 8 bits
* :func:`rms_norm_fp8` – residual's addition, root-mean-square norm and conversion in one pass
* :func:`matmul_fp8` – the product of such rows with such weights, of one matrix or of many experts
* :func:`moe_few_tokens` – a whole SwiGLU mixture-of-experts layer for up to 64 tokens

CUDA tensors run on the native kernels, on the current stream of their device; CPU tensors on
the plain statements in :mod:`lplb_b200.ops.reference`.  Calls can be captured in a CUDA graph.  None has a
backward pass; an argument that requires a gradient is refused.  Wrong arguments raise
``ValueError``.  :func:`check` returns the first error that a kernel has seen.

The reference has no operators of this kind.
"""

from __future__ import annotations

import torch

from . import reference

__all__ = [
    "MOE_FEW_MAX_EXPERTS",
    "MOE_FEW_MAX_HIDDEN",
    "MOE_FEW_MAX_INTER",
    "MOE_FEW_MAX_TOKENS",
    "MOE_FEW_MAX_TOPK",
    "quantize_fp8",
    "quantize_weight_fp8",
    "rms_norm_fp8",
    "matmul_fp8",
    "moe_few_tokens",
    "check",
]


MOE_FEW_MAX_TOKENS = 64  #: tokens that moe_few_tokens takes
MOE_FEW_MAX_TOPK, MOE_FEW_MAX_EXPERTS, MOE_FEW_MAX_HIDDEN, MOE_FEW_MAX_INTER = 32, 512, 16384, 65536  # and the rest of its range

_module = None


def _native():
    global _module
    if _module is None:
        from .. import _native

        _module = _native.load()
    return _module


def _need(ok: bool, message: str) -> None:
    """Refusals of CPU arguments, in the words of the native binding."""
    if not ok:
        raise ValueError(f"lplb_b200.ops.{message}")


def _check_type(x: torch.Tensor, who: str) -> None:
    _need(x.dtype in (torch.float32, torch.bfloat16, torch.float16), f"{who} must be float32, bfloat16 or float16, not {x.dtype}")


def _check_device(who: str, first: torch.Tensor, *others: torch.Tensor | None) -> None:
    _need(all(t is None or t.device == first.device for t in others), f"{who} all arguments must be on one device")


def _check_rows(x: torch.Tensor, who: str) -> None:
    _check_type(x, who)
    _need(x.dim() >= 1 and 1 <= x.shape[-1] <= 16384, f"{who} must have rows of 1 to 16384 values")
    _check_no_grad(x, who)


def _check_no_grad(x: torch.Tensor, who: str) -> None:
    _need(not (x.requires_grad and torch.is_grad_enabled()), f"{who} requires a gradient: these operators have no backward pass")


def quantize_fp8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``(q, scale)`` of rows ``x`` ``[..., K]`` (float32, bfloat16 or float16; rows may be apart from one
    another): ``q`` ``[..., K]`` and one scale per 128, ``[..., ceil(K / 128)]``, both contiguous."""
    if x.is_cuda:
        return _native().quantize_fp8(x)
    _check_rows(x, "quantize_fp8: x")
    return reference.quantize_fp8_reference(x)


def quantize_weight_fp8(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``(q, scale)`` of contiguous weights ``[N, K]`` or ``[E, N, K]`` (float32, bfloat16 or float16): one scale per 128 x 128,
    ``[..., ceil(N / 128), ceil(K / 128)]``."""
    if w.is_cuda:
        return _native().quantize_weight_fp8(w)
    _need(w.dim() in (2, 3) and w.is_contiguous(), "quantize_weight_fp8: w must be contiguous [rows, cols] or [matrices, rows, cols]")
    _check_type(w, "quantize_weight_fp8: w")
    _check_no_grad(w, "quantize_weight_fp8: w")
    return reference.quantize_weight_fp8_reference(w)


def rms_norm_fp8(
    x: torch.Tensor,
    weight: torch.Tensor,
    residual: torch.Tensor | None = None,
    eps: float = 1e-6,
    return_normed: bool = False,
) -> tuple[torch.Tensor, ...]:
    """``(q, scale, h)`` with ``h = x + residual`` rounded to ``x``'s type and ``(q, scale)`` the 8-bit form
    of ``h / sqrt(mean(h**2) + eps) * weight`` over the last dimension, computed in 32 bits.  Without a
    residual ``h`` is ``x`` itself.  ``weight`` is of ``x``'s type or float32.  ``return_normed`` adds the
    normed rows in ``x``'s type, which a router reads."""
    if x.is_cuda:
        return _native().rms_norm_fp8(x, weight, residual, eps, return_normed)
    _check_rows(x, "rms_norm_fp8: x")
    _check_device("rms_norm_fp8:", x, weight, residual)
    _check_no_grad(weight, "rms_norm_fp8: weight")
    _need(weight.shape == x.shape[-1:], "rms_norm_fp8: weight must have one value for each of a row")
    _need(weight.dtype in (x.dtype, torch.float32), "rms_norm_fp8: weight must be float32 or of x's type")
    _need(eps >= 0, "rms_norm_fp8: eps must not be negative")
    if residual is not None:
        _check_rows(residual, "rms_norm_fp8: residual")
        _need(residual.shape == x.shape and residual.dtype == x.dtype, "rms_norm_fp8: residual must have x's shape and type")
    return reference.rms_norm_fp8_reference(x, weight, residual, eps, return_normed)


def matmul_fp8(
    a: torch.Tensor,
    a_scale: torch.Tensor,
    b: torch.Tensor,
    b_scale: torch.Tensor,
    rows: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
    out_dtype: torch.dtype = torch.bfloat16,
    status: torch.Tensor | None = None,
) -> torch.Tensor:
    """``a @ b.T`` of the values that ``a`` ``[M, K]`` (scales ``[M, ceil(K / 128)]``) and ``b`` ``[N, K]``
    (scales ``[ceil(N / 128), ceil(K / 128)]``) stand for, summed in 32 bits, in bfloat16 or float32.

    With ``rows`` (int32 ``[E]``, on ``a``'s device, E up to 128) ``b`` is ``[E, N, K]`` and its matrix ``e`` takes
    ``rows[e]`` rows of ``a``, which follow those of matrix ``e - 1``; no more rows are taken than ``a`` has.  Rows behind
    the last group are left in ``out`` as they were (in a new ``out``: not set).

    ``K`` is a multiple of 16; ``a``, and all matrices of ``b`` together, have up to 2**31 - 256 rows.  Rows of ``a``, of
    ``a_scale`` and of ``out`` may be apart from one another; those of ``a`` start on 16-byte boundaries, as does ``b``, which is
    contiguous with its scales.  ``status``: see :func:`check`."""
    if out_dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"lplb_b200.ops.matmul_fp8: out_dtype must be bfloat16 or float32, not {out_dtype}")
    if a.is_cuda:
        return _native().matmul_fp8(a, a_scale, b, b_scale, rows, out, out_dtype == torch.float32, status)
    _check_device("matmul_fp8:", a, a_scale, b, b_scale, rows, out)
    e4m3, e8m0, lead = torch.float8_e4m3fn, torch.float8_e8m0fnu, 0 if rows is None else 1
    _need(a.dim() == 2 and a.dtype == e4m3, "matmul_fp8: a must be [rows, k] of float8_e4m3fn")
    _need(b.dim() == 2 + lead and b.dtype == e4m3, "matmul_fp8: b must be [n, k] (with rows: [groups, n, k]) of float8_e4m3fn")
    m, k, n, blocks = *a.shape, b.shape[-2], -(-a.shape[1] // 128)
    most = 2**31 - 256
    _need(m <= most and n * (b.shape[0] if lead else 1) <= most, f"matmul_fp8: at most {most} rows of a, and of all matrices of b together")
    _need(k >= 16 and k % 16 == 0 and b.shape[-1] == k, "matmul_fp8: a and b must have the same k, a multiple of 16")
    _need(a_scale.dtype == e8m0 and a_scale.shape == (m, blocks), "matmul_fp8: a_scale must be [rows, ceil(k / 128)]")
    _need(
        b_scale.dtype == e8m0 and b_scale.shape == (*b.shape[:lead], -(-n // 128), blocks),
        "matmul_fp8: b_scale must be [ceil(n / 128), ceil(k / 128)] (with rows: for every group)",
    )
    _need(rows is None or (rows.dtype == torch.int32 and rows.shape == b.shape[:1]), "matmul_fp8: rows must be int32, one for each matrix")
    _need(rows is None or b.shape[0] <= 128, "matmul_fp8: 1 to 128 groups")
    _need(out is None or (out.shape == (m, n) and out.dtype == out_dtype), "matmul_fp8: out must be [rows, n] of the output type")
    if out is not None:
        _check_no_grad(out, "matmul_fp8: out")
    result = reference.matmul_fp8_reference(a, a_scale, b, b_scale, rows).to(out_dtype)
    if out is None:
        return result
    taken = m if rows is None else min(m, int(rows.clamp_min(0).sum()))
    out[:taken] = result[:taken]
    return out


def moe_few_tokens(
    x: torch.Tensor,
    idx: torch.Tensor,
    weights: torch.Tensor,
    w13: torch.Tensor,
    w2: torch.Tensor,
    x_scale: torch.Tensor | None = None,
    w13_scale: torch.Tensor | None = None,
    w2_scale: torch.Tensor | None = None,
    status: torch.Tensor | None = None,
) -> torch.Tensor:
    """A whole SwiGLU mixture-of-experts layer for up to 64 tokens: two kernels that read the weights of the
    chosen experts once.

    ``out[t] = sum_k weights[t, k] * (silu(x[t] @ gate.T) * (x[t] @ up.T)) @ down.T`` of expert ``idx[t, k]``, bfloat16
    ``[tokens, hidden]``.  ``idx`` ``[tokens, topk]`` (int64 or int32) holds physical ids; -1 and ids that no expert has
    choose nothing, an expert chosen twice counts twice.  ``w13`` ``[experts, 2 * inter, hidden]`` is laid out in
    blocks of 128 gate rows and their 128 up rows (``lplb_b200.models.interleave_gate_up``), ``w2`` is ``[experts,
    hidden, inter]``; ``hidden`` is a multiple of 256 up to 16384, ``inter`` of 128 up to 65536; up to 512 experts and 32 choices per token.

    bfloat16 weights take bfloat16 ``x`` and hold the activations in bfloat16.  Weights in 8 bits (``w13_scale``,
    ``w2_scale`` as :func:`quantize_weight_fp8` gives them) take ``x`` in 8 bits with its ``x_scale``, or in bfloat16,
    which the first kernel converts, and hold the activations in 8 bits with a scale per 128.  Sums are in 32 bits
    throughout, over experts too; the same inputs give the same bits.  ``status``: see :func:`check`."""
    if x.is_cuda:
        return _native().moe_few_tokens(x, idx, weights, w13, w2, x_scale, w13_scale, w2_scale, status)
    fp8, who = w13_scale is not None, "moe_few_tokens:"
    _check_device(who, x, idx, weights, w13, w2, x_scale, w13_scale, w2_scale)
    _need(x.dim() == 2 and x.shape[0] <= MOE_FEW_MAX_TOKENS, f"{who} at most {MOE_FEW_MAX_TOKENS} tokens")
    _need(fp8 == (w2_scale is not None), f"{who} w13_scale and w2_scale come together")
    _need(fp8 or x_scale is None, f"{who} x_scale needs weights in 8 bits")
    wtype = torch.float8_e4m3fn if fp8 else torch.bfloat16
    _need(w13.dim() == 3 and w2.dim() == 3 and w13.dtype == wtype and w2.dtype == wtype, f"{who} w13 and w2 must be {wtype}")
    experts, inter, hidden = w13.shape[0], w13.shape[1] // 2, x.shape[1]
    _need(
        hidden % 256 == 0 and 0 < hidden <= MOE_FEW_MAX_HIDDEN and inter % 128 == 0 and 0 < inter <= MOE_FEW_MAX_INTER,
        f"{who} hidden must be a multiple of 256 (up to {MOE_FEW_MAX_HIDDEN}), inter of 128 (up to {MOE_FEW_MAX_INTER})",
    )
    _need(
        w13.shape == (experts, 2 * inter, hidden) and w2.shape == (experts, hidden, inter),
        f"{who} w13 must be [experts, 2 * inter, hidden], w2 [experts, hidden, inter]",
    )
    _need(1 <= experts <= MOE_FEW_MAX_EXPERTS, f"{who} 1 to {MOE_FEW_MAX_EXPERTS} experts")
    _need(x.dtype == (torch.bfloat16 if x_scale is None else torch.float8_e4m3fn), f"{who} x must be bfloat16, or float8_e4m3fn with x_scale")
    _need(idx.dim() == 2 and idx.shape[0] == x.shape[0] and idx.dtype in (torch.int64, torch.int32), f"{who} idx must be [tokens, topk]")
    _need(1 <= idx.shape[1] <= MOE_FEW_MAX_TOPK, f"{who} 1 to {MOE_FEW_MAX_TOPK} choices per token")
    _need(weights.shape == idx.shape and weights.is_floating_point(), f"{who} weights must be floating point, of idx's shape")
    for scale in (x_scale, w13_scale, w2_scale):
        _need(scale is None or scale.dtype == torch.float8_e8m0fnu, f"{who} scales must be float8_e8m0fnu")
    for scale, of in ((w13_scale, w13), (w2_scale, w2)):
        _need(scale is None or scale.shape == (experts, of.shape[1] // 128, of.shape[2] // 128), f"{who} scales must be [experts, rows / 128, cols / 128]")
    _need(x_scale is None or x_scale.shape == (x.shape[0], hidden // 128), f"{who} x_scale must be [tokens, hidden / 128]")
    for t in (x, weights, w13, w2):
        _check_no_grad(t, f"{who} an argument")
    return reference.moe_few_tokens_reference(x, idx, weights, w13, w2, x_scale, w13_scale, w2_scale).bfloat16()


def check(device: torch.device | int | None = None, clear: bool = False) -> int:
    """First error code that a kernel of these operators has raised on ``device`` (0: none; 21: a wait inside
    a kernel gave up, its results are not valid).  Waits for the device; ``clear`` forgets the error.

    A call that is given ``status``, an int32 tensor on its device, leaves its first error in that tensor's first word (where that is
    0) and not here: callers that keep their errors apart, as ``MoELayer`` does."""
    index = torch.device("cuda" if device is None else device).index if not isinstance(device, int) else device
    return _native().ops_error(torch.cuda.current_device() if index is None else index, clear)

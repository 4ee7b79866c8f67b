"""The product with an epilogue in 16 bits, for training and serving: of one matrix, or of many experts' rows."""

from __future__ import annotations

import torch

from . import reference
from .experts import _first_order, _wants_grad
from .fp8 import _check_device, _native, _need

__all__ = ["MATMUL_ACTIVATIONS", "MATMUL_MAX_GROUPS", "matmul"]

MATMUL_ACTIVATIONS = (None, "relu", "gelu", "silu", "swiglu")  #: what matmul takes for ``activation``
MATMUL_MAX_GROUPS = 1024  #: matrices that matmul takes with ``rows``

_MOST_ROWS = 2**31 - 256


class _Matmul(torch.autograd.Function):
    """On the CPU."""

    @staticmethod
    def forward(ctx, a, b, bias, residual, rows, activation, out_dtype):
        out, z = reference.matmul_reference(a, b, bias, activation, residual, rows)
        ctx.save_for_backward(a, b, rows, z if activation is not None else None)
        ctx.options = activation, None if bias is None else bias.dtype
        return out.to(out_dtype)

    @staticmethod
    @_first_order
    def backward(ctx, dout):
        a, b, rows, z = ctx.saved_tensors
        activation, bias_dtype = ctx.options
        need_a, need_b, need_bias, need_residual = ctx.needs_input_grad[:4]
        da, db, dbias = reference.matmul_backward_reference(dout, a, b, z, activation, rows)
        return (
            da.to(a.dtype) if need_a else None,
            db.to(b.dtype) if need_b else None,
            dbias.to(bias_dtype) if need_bias else None,
            dout if need_residual else None,
            None,
            None,
            None,
        )


def matmul(
    a: torch.Tensor,
    b: torch.Tensor,
    bias: torch.Tensor | None = None,
    activation: str | None = None,
    residual: torch.Tensor | None = None,
    rows: torch.Tensor | None = None,
    out_dtype: torch.dtype | None = None,
) -> torch.Tensor:
    """``act(a @ b.T + bias) + residual`` for ``a`` ``[M, K]`` and weights ``b`` ``[N, K]``, both bfloat16 or both float16,
    summed in 32 bits and rounded once, to ``out_dtype``: ``a``'s type (default) or float32.

    ``activation`` is None, ``"relu"``, ``"gelu"`` (``z`` times the normal distribution's function), ``"silu"`` or ``"swiglu"``,
    ``silu(gate) * up`` of ``N / 2`` columns, for which ``b`` (and ``bias``) lies in blocks of 128 gate rows and their 128 up rows
    (``lplb_b200.models.interleave_gate_up``).  ``bias`` ``[N]`` is of ``a``'s type or float32, ``residual`` of the output's shape
    and type.

    With ``rows`` (int32 ``[E]`` on ``a``'s device, E up to 1024; ``counts`` of :func:`~lplb_b200.ops.expert_order`) ``b`` is
    ``[E, N, K]`` and ``bias`` ``[E, N]``; matrix ``e`` takes ``rows[e]`` rows of ``a``, which follow those of matrix ``e - 1``; no
    more rows are taken than ``a`` has, negative numbers take none.  Rows behind the last group have no product: they are the
    residual's, or zero.

    ``K`` is a multiple of 8; ``a``, and all matrices of ``b`` together, have up to 2**31 - 256 rows.  ``b`` is contiguous and starts
    on a 16-byte boundary; rows of ``a`` that do not are copied first.

    Differentiable with respect to ``a``, ``b``, ``bias`` and ``residual``; a gradient's gradient is refused, and so is a CUDA tensor with
    a forward-mode tangent.  For the backward pass the sums before an activation are kept, in 32 bits, and their gradients are rounded
    to ``a``'s bits before they are multiplied: to bfloat16, or to the 11 bits of float16 in parts of a power of two, so that what
    float16 does not hold on the way, large or small, is not lost.  All sums are in 32 bits.

    CUDA tensors run on the native kernels, on the current stream of their device, CPU tensors on plain statements; calls and
    backward passes can be captured in a CUDA graph, and the same inputs give the same bits.  Inside a capture a call that is
    recorded is refused (``RuntimeError``) while a graph recorded on the default stream still holds one of its leaves: delete that
    graph's outputs first, or call under ``torch.no_grad()`` if there will be no backward pass.  Wrong arguments raise
    ``ValueError``; :func:`~lplb_b200.ops.check` tells of waits that ran out."""
    if activation not in MATMUL_ACTIVATIONS:  # (messages are put together where they are needed: the call is a few microseconds)
        raise ValueError(f"lplb_b200.ops.matmul: activation must be one of {MATMUL_ACTIVATIONS}, not {activation!r}")
    if out_dtype is None:
        out_dtype = a.dtype
    elif out_dtype is not torch.float32 and out_dtype is not a.dtype:
        raise ValueError(f"lplb_b200.ops.matmul: out_dtype must be a's type or float32, not {out_dtype}")
    if a.is_cuda:
        return _native().matmul(a, b, bias, MATMUL_ACTIVATIONS.index(activation), residual, rows, out_dtype is torch.float32)
    _check(a, b, bias, activation, residual, rows, out_dtype, "matmul:")
    if _wants_grad(a, b, bias, residual):
        return _Matmul.apply(a, b, bias, residual, rows, activation, out_dtype)
    return reference.matmul_reference(a, b, bias, activation, residual, rows)[0].to(out_dtype)


def _check(a, b, bias, activation, residual, rows, out_dtype, who):
    """Refusals of CPU arguments, as the native binding's."""
    _check_device(who, a, b, bias, residual, rows)
    lead = 0 if rows is None else 1
    _need(a.dim() == 2 and a.dtype in (torch.bfloat16, torch.float16), f"{who} a must be [rows, k] of bfloat16 or float16")
    _need(b.dim() == 2 + lead and b.dtype == a.dtype, f"{who} b must be [n, k] (with rows: [groups, n, k]) of a's type")
    m, k, n, groups = *a.shape, b.shape[-2], b.shape[0] if lead else 1
    _need(1 <= groups <= MATMUL_MAX_GROUPS, f"{who} 1 to {MATMUL_MAX_GROUPS} groups")
    _need(rows is None or (rows.dtype == torch.int32 and rows.shape == (groups,)), f"{who} rows must be int32, one number for each matrix of b")
    _need(m <= _MOST_ROWS and groups * n <= _MOST_ROWS, f"{who} at most {_MOST_ROWS} rows of a, and of all matrices of b together")
    _need(8 <= k <= 2**28 and k % 8 == 0 and b.shape[-1] == k, f"{who} a and b must have the same k, a multiple of 8")
    _need(1 <= n <= 2**28, f"{who} b has no rows, or too many")
    _need(b.is_contiguous() and b.data_ptr() % 16 == 0, f"{who} b must be contiguous and start on a 16-byte boundary")
    _need(activation != "swiglu" or n % 256 == 0, f"{who} 'swiglu' needs blocks of 128 gate rows and their 128 up rows: n must be a multiple of 256")
    _need(
        bias is None or (bias.dtype in (a.dtype, torch.float32) and bias.shape == b.shape[:-1]),
        f"{who} bias must be [n] (with rows: [groups, n]) of a's type or float32",
    )
    cols = n // 2 if activation == "swiglu" else n
    _need(residual is None or (residual.dtype == out_dtype and residual.shape == (m, cols)), f"{who} residual must be of the output's shape and type")

"""Operators around a layer's experts in 16 and 32 bits, for training and serving.

* :func:`gate_topk` – a router's logits to the chosen experts and their weights
* :func:`expert_order` – which row every choice has once the rows are sorted by expert
* :func:`take_rows` – the tokens' rows in that order
* :func:`combine_rows` – the experts' rows back to their tokens, weighted

Between the last two stand the experts' products: :func:`lplb_b200.ops.matmul` with ``rows=order.counts`` (or, for rows in 8
bits, ``matmul_fp8``)::

    weights, logical_idx = ops.gate_topk(logits, 8)
    order = ops.expert_order(planner.run(logical_idx, avail), planner.n_routed_experts)
    rows = ops.take_rows(x, order)
    act = ops.matmul(rows, w13, activation="swiglu", rows=order.counts)
    y = ops.combine_rows(ops.matmul(act, w2, rows=order.counts), order, weights)

Every one but :func:`expert_order`, which has whole numbers alone, has a gradient; a gradient's gradient is refused, and so is a CUDA
tensor with a forward-mode tangent.  CUDA tensors run on the native kernels, on the current stream of their device; CPU tensors on
the plain statements in :mod:`lplb_b200.ops.reference`.  Calls can be captured in a CUDA graph, backward passes too; inside a capture
a call that is recorded is refused (``RuntimeError``) while a graph recorded on the default stream still holds one of its leaves.
The same inputs give the same bits.  Wrong arguments raise ``ValueError``.

The reference has no operators of this kind.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import reference
from .fp8 import _check_device, _check_type, _native, _need

__all__ = ["GATE_MAX_EXPERTS", "GATE_MAX_TOPK", "ORDER_MAX_EXPERTS", "ExpertOrder", "gate_topk", "expert_order", "take_rows", "combine_rows"]

GATE_MAX_EXPERTS, GATE_MAX_TOPK = 1024, 32  #: experts and choices that gate_topk takes
ORDER_MAX_EXPERTS = 1024  #: experts that expert_order takes

_MOST_VALUES = (2**31 - 1) // 16  # of a row


def _whole(n, who: str) -> int:
    """``n`` as a whole number, which nothing is cut off to make."""
    if type(n) is int and -(2**62) < n < 2**62:
        return n
    try:
        whole = int(n)
        if whole == n and -(2**63) <= whole < 2**63:
            return whole
    except (TypeError, ValueError, OverflowError):
        pass
    raise ValueError(f"lplb_b200.ops.{who} must be a whole number, not {n!r}")


def _wants_grad(*tensors: torch.Tensor | None) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _first_order(backward):
    """For a backward pass on the CPU: its gradients refuse to be differentiated, as the native ones do."""

    def wrapped(ctx, *grads):
        with torch.no_grad():
            found = backward(ctx, *grads)
        if not torch.is_grad_enabled():
            return found
        leaves = [g.detach().requires_grad_() for g in found if g is not None]
        refuse = torch._C._functions.DelayedError(b"lplb_b200.ops: a gradient's gradient is not computed", len(leaves))
        marked = iter(refuse(*leaves) if len(leaves) > 1 else (refuse(*leaves),)) if leaves else iter(())
        return tuple(None if g is None else next(marked) for g in found)

    return wrapped


# ---------------------------------------------------------------------------------- the router's choice
class _GateTopk(torch.autograd.Function):
    """On the CPU."""

    @staticmethod
    def forward(ctx, logits, topk, score, renormalize, scale):
        weights, idx = reference.gate_topk_reference(logits, topk, score, renormalize, scale)
        ctx.save_for_backward(logits, idx)
        ctx.mark_non_differentiable(idx)
        ctx.options = score, renormalize, scale
        return weights, idx

    @staticmethod
    @_first_order
    def backward(ctx, dweights, _):
        logits, idx = ctx.saved_tensors
        return reference.gate_topk_backward_reference(logits, idx, dweights, *ctx.options), None, None, None, None


def gate_topk(
    logits: torch.Tensor, topk: int, score: str = "softmax", renormalize: bool = False, scale: float = 1.0
) -> tuple[torch.Tensor, torch.Tensor]:
    """``(weights, idx)``, float32 and int64 ``[tokens, topk]``: for every token the ``topk`` largest of its ``logits``
    ``[tokens, experts]`` (float32, bfloat16 or float16), largest first, of equal ones the lower expert first, and their weights
    ``scale * s[idx]`` with the scores ``s = softmax(logits)`` or ``sigmoid(logits)``.  ``renormalize`` divides a token's
    weights, before the scale, by their sum.

    A logit of -infinity is an expert that cannot be chosen: where fewer than ``topk`` are left, ``idx`` is -1, which the planner and
    :func:`expert_order` take for no choice, and the weight is 0.  A NaN counts as larger than any number and makes the weights that
    depend on it NaN.  Up to 1024 experts and 32 choices.  Differentiable with respect to ``logits``."""
    if score not in ("softmax", "sigmoid"):
        raise ValueError(f"lplb_b200.ops.gate_topk: score must be 'softmax' or 'sigmoid', not {score!r}")
    topk = _whole(topk, "gate_topk: topk")
    if logits.is_cuda:
        return _native().gate_topk(logits, topk, score == "sigmoid", bool(renormalize), float(scale))
    who, renormalize, scale = "gate_topk:", bool(renormalize), float(scale)
    _check_type(logits, f"{who} logits")
    _need(logits.dim() == 2, f"{who} logits must be [tokens, experts]")
    _need(1 <= logits.shape[1] <= GATE_MAX_EXPERTS, f"{who} 1 to {GATE_MAX_EXPERTS} experts")
    _need(logits.shape[0] < 2**31, f"{who} fewer than 2^31 tokens")
    _need(1 <= topk <= min(GATE_MAX_TOPK, logits.shape[1]), f"{who} topk must be 1 to {GATE_MAX_TOPK}, and no more than there are experts")
    if _wants_grad(logits):
        return _GateTopk.apply(logits, topk, score, renormalize, scale)
    return reference.gate_topk_reference(logits, topk, score, renormalize, scale)


# ---------------------------------------------------------------------------------- rows sorted by expert
class ExpertOrder(NamedTuple):
    """Where the rows of a batch's choices are once they are sorted by expert."""

    counts: torch.Tensor  #: int32 ``[experts]``, rows of every expert: ``rows`` of :func:`~lplb_b200.ops.matmul` and ``matmul_fp8``
    place: torch.Tensor  #: int32 ``[tokens, topk]``, the row of every choice, or -1
    source: torch.Tensor  #: int32 ``[tokens * topk]``, the choice (token * topk + k) of every row, or -1 behind the last


def expert_order(idx: torch.Tensor, n_experts: int) -> ExpertOrder:
    """The order of rows by expert, within an expert by token and choice, of ``idx`` ``[tokens, topk]`` (int64 or int32: a
    gate's experts, or physical ones as the planner gives them).  Numbers outside ``[0, n_experts)``, -1 among them, choose
    nothing.  Up to 1024 experts and 1024 choices per token, fewer than 2**31 choices in all.  Nothing waits for the device:
    there are as many rows as choices, and those behind the last expert's are nobody's."""
    n_experts = _whole(n_experts, "expert_order: n_experts")
    if idx.is_cuda:
        return ExpertOrder(*_native().expert_order(idx, n_experts))
    who = "expert_order:"
    _need(idx.dim() == 2 and idx.dtype in (torch.int64, torch.int32), f"{who} idx must be [tokens, topk] of int64 or int32")
    _need(1 <= n_experts <= ORDER_MAX_EXPERTS, f"{who} 1 to {ORDER_MAX_EXPERTS} experts")
    _need(1 <= idx.shape[1] <= 1024, f"{who} 1 to 1024 choices per token")
    _need(idx.numel() < 2**31, f"{who} fewer than 2^31 choices in all")
    return ExpertOrder(*reference.expert_order_reference(idx, n_experts))


def _check_order(rows: torch.Tensor, order: ExpertOrder, who: str) -> None:
    _check_device(who, rows, order.place, order.source)
    _need(
        order.place.dim() == 2 and order.place.dtype == torch.int32 and order.place.shape[1] >= 1
        and order.source.dtype == torch.int32 and order.source.shape == (order.place.numel(),),
        f"{who} order must be one of expert_order's",
    )


class _TakeRows(torch.autograd.Function):
    """On the CPU."""

    @staticmethod
    def forward(ctx, x, place, source):
        ctx.save_for_backward(place)
        return reference.take_rows_reference(x, place, source)

    @staticmethod
    @_first_order
    def backward(ctx, drows):
        return reference.combine_rows_reference(drows, *ctx.saved_tensors), None, None


class _CombineRows(torch.autograd.Function):
    """On the CPU."""

    @staticmethod
    def forward(ctx, rows, weights, place, source):
        ctx.save_for_backward(*((place, source) if weights is None else (place, source, rows, weights)))
        return reference.combine_rows_reference(rows, place, weights)

    @staticmethod
    @_first_order
    def backward(ctx, dout):
        place, source, *kept = ctx.saved_tensors
        if not kept:
            return reference.take_rows_reference(dout, place, source), None, None, None
        drows, dweights = reference.combine_rows_backward_reference(dout, kept[0], place, kept[1])
        need_rows, need_weights = ctx.needs_input_grad[:2]
        return drows if need_rows else None, dweights if need_weights else None, None, None


def take_rows(x: torch.Tensor, order: ExpertOrder) -> torch.Tensor:
    """``rows`` ``[tokens * topk, values]``, contiguous: ``rows[order.place[t, k]] = x[t]``; rows behind the last
    expert's are zero.  ``x`` is ``[tokens, values]`` of any type, values in 8 bits and their scales among them, of up to (2**31 - 1) //
    16 values; rows may be apart from one another.  Differentiable for float32, bfloat16 and float16: ``dx[t]`` is the sum of its
    rows' gradients, in 32 bits."""
    if x.is_cuda:
        return _native().take_rows(x, order.place, order.source)
    _need(x.dim() == 2, "take_rows: x must be [tokens, values]")
    _need(1 <= x.shape[1] <= _MOST_VALUES, "take_rows: rows without values, or too long")
    _check_order(x, order, "take_rows:")
    _need(order.place.shape[0] == x.shape[0], "take_rows: x must have a row for each of the order's tokens")
    if _wants_grad(x):
        _check_type(x, "take_rows: x that requires a gradient")
        return _TakeRows.apply(x, order.place, order.source)
    return reference.take_rows_reference(x, order.place, order.source)


def combine_rows(rows: torch.Tensor, order: ExpertOrder, weights: torch.Tensor | None = None) -> torch.Tensor:
    """``out[t] = sum over k of weights[t, k] * rows[order.place[t, k]]`` ``[tokens, values]`` of the rows' type (float32,
    bfloat16 or float16), summed in 32 bits in the order of ``k`` and rounded once; without ``weights`` the plain sum.  ``rows`` is
    ``[tokens * topk, values]``; choices without a row add nothing, and rows behind the last expert's are not read.  ``weights``
    ``[tokens, topk]`` is of any floating type and used in 32 bits.  Differentiable with respect to ``rows`` (zero where a row is
    nobody's) and ``weights`` (zero where a choice has no row)."""
    if rows.is_cuda:
        return _native().combine_rows(rows, order.place, order.source, weights)
    who = "combine_rows:"
    _check_type(rows, f"{who} rows")
    _need(rows.dim() == 2, f"{who} rows must be [tokens * topk, values]")
    _need(1 <= rows.shape[1] <= _MOST_VALUES, f"{who} rows without values, or too long")
    _check_device(who, rows, weights)
    _check_order(rows, order, who)
    _need(rows.shape[0] == order.place.numel(), f"{who} rows must have one for each of the order's choices")
    _need(weights is None or (weights.is_floating_point() and weights.shape == order.place.shape), f"{who} weights must be floating point [tokens, topk]")
    weights = None if weights is None else weights.float()
    if _wants_grad(rows, weights):
        return _CombineRows.apply(rows, weights, order.place, order.source)
    return reference.combine_rows_reference(rows, order.place, weights)

"""Operators: plain PyTorch statements of the planner's kernels (the numerics oracles and the CPU path), the
8-bit serving operators that stand around a mixture-of-experts layer, and the operators around and inside its experts in
16 and 32 bits, with their gradients."""

from . import reference
from .dense import MATMUL_ACTIVATIONS, MATMUL_MAX_GROUPS, matmul
from .experts import (
    GATE_MAX_EXPERTS,
    GATE_MAX_TOPK,
    ORDER_MAX_EXPERTS,
    ExpertOrder,
    combine_rows,
    expert_order,
    gate_topk,
    take_rows,
)
from .fp8 import (
    MOE_FEW_MAX_EXPERTS,
    MOE_FEW_MAX_HIDDEN,
    MOE_FEW_MAX_INTER,
    MOE_FEW_MAX_TOKENS,
    MOE_FEW_MAX_TOPK,
    check,
    matmul_fp8,
    moe_few_tokens,
    quantize_fp8,
    quantize_weight_fp8,
    rms_norm_fp8,
)
from .reference import (
    count_reference,
    dequantize_fp8,
    dequantize_weight_fp8,
    quotas_reference,
    redirect_reference,
    slice_bounds,
)

__all__ = [
    "MOE_FEW_MAX_EXPERTS",
    "MOE_FEW_MAX_HIDDEN",
    "MOE_FEW_MAX_INTER",
    "MOE_FEW_MAX_TOKENS",
    "MOE_FEW_MAX_TOPK",
    "reference",
    "count_reference",
    "quotas_reference",
    "redirect_reference",
    "slice_bounds",
    "quantize_fp8",
    "quantize_weight_fp8",
    "dequantize_fp8",
    "dequantize_weight_fp8",
    "rms_norm_fp8",
    "matmul_fp8",
    "moe_few_tokens",
    "check",
    "GATE_MAX_EXPERTS",
    "GATE_MAX_TOPK",
    "ORDER_MAX_EXPERTS",
    "ExpertOrder",
    "gate_topk",
    "expert_order",
    "take_rows",
    "combine_rows",
    "MATMUL_ACTIVATIONS",
    "MATMUL_MAX_GROUPS",
    "matmul",
]

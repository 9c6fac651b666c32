"""MI355X-native INT8 "convrot" linear for HyperFlow H3 Flash: a drop-in for ``hyperflow_h3_flash.int8``, and the
operators of an attention block around it (norms and rotation, packed attention, adapters of many requests).

Importing the package does not touch the GPU or load the HIP library; the first device forward does.
"""

from .attention_block import AdapterBank, AttentionBlock
from .block import AdapterPlan, AttentionPlan, RotaryAxes, adapter_add, packed_attention, qk_norm_rope
from .int8 import (
    ACTIVATIONS,
    ARITHMETIC_OPTIONS,
    INT8_GEMMS,
    KERNEL_OPTIONS,
    ROTATE_ARITHMETICS,
    ROTATE_QUANTS,
    Int8RotLinear,
    hadamard_factors,
    regular_hadamard,
    resolve_int8_gemm,
    set_arithmetic_options,
    set_kernel_options,
)
from .lowrank import RANK_MULTIPLE, LowRankLinear, fuse_qkv, set_lowrank_rank_multiple

__version__ = "0.1.0"

__all__ = [
    "ACTIVATIONS",
    "ARITHMETIC_OPTIONS",
    "AdapterBank",
    "AdapterPlan",
    "AttentionBlock",
    "AttentionPlan",
    "INT8_GEMMS",
    "KERNEL_OPTIONS",
    "ROTATE_ARITHMETICS",
    "ROTATE_QUANTS",
    "Int8RotLinear",
    "LowRankLinear",
    "RANK_MULTIPLE",
    "RotaryAxes",
    "adapter_add",
    "fuse_qkv",
    "hadamard_factors",
    "packed_attention",
    "qk_norm_rope",
    "regular_hadamard",
    "resolve_int8_gemm",
    "set_arithmetic_options",
    "set_kernel_options",
    "set_lowrank_rank_multiple",
]

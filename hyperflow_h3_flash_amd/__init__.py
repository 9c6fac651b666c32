"""MI355X-native INT8 "convrot" linear for HyperFlow H3 Flash: a drop-in for ``hyperflow_h3_flash.int8``, and the
operators of a transformer block around it (norms and rotation, packed attention, adapters of many requests, keys and values
held in 4 bits, norms with gates and residuals).

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
from .kv_cache import CachePlan, KVCache, cache_append, cache_read, cached_attention, copy_pages
from .lowrank import RANK_MULTIPLE, LowRankLinear, fuse_qkv, set_lowrank_rank_multiple
from .residual_norm import RowPlan, residual_norm
from .transformer_block import TransformerBlock, TransformerStack

__version__ = "0.1.0"

__all__ = [
    "ACTIVATIONS",
    "ARITHMETIC_OPTIONS",
    "AdapterBank",
    "AdapterPlan",
    "AttentionBlock",
    "AttentionPlan",
    "CachePlan",
    "INT8_GEMMS",
    "KERNEL_OPTIONS",
    "ROTATE_ARITHMETICS",
    "ROTATE_QUANTS",
    "Int8RotLinear",
    "KVCache",
    "LowRankLinear",
    "RANK_MULTIPLE",
    "RotaryAxes",
    "RowPlan",
    "TransformerBlock",
    "TransformerStack",
    "adapter_add",
    "cache_append",
    "cache_read",
    "cached_attention",
    "copy_pages",
    "fuse_qkv",
    "hadamard_factors",
    "packed_attention",
    "qk_norm_rope",
    "regular_hadamard",
    "residual_norm",
    "resolve_int8_gemm",
    "set_arithmetic_options",
    "set_kernel_options",
    "set_lowrank_rank_multiple",
]

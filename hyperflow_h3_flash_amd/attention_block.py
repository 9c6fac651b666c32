"""An attention block around the INT8 linears, for several requests packed in one batch.

`AttentionBlock` runs the fused q/k/v projection, each request's adapters beside it, the norms and rotation of queries
and keys, attention within each request, and the output projection with its adapters; `AdapterBank` holds the adapters of
one projection. The reference's blocks do the same between ``to_q``/``to_k``/``to_v`` and ``to_out``
(src/hyperflow_h3_flash/transformer.py:339-380), for one request and without adapters."""

from __future__ import annotations

import warnings

import torch
from torch import Tensor, nn

from .block import (AdapterPlan, AttentionPlan, RotaryAxes, _differentiable, _forward_only, adapter_add, packed_attention,
                    qk_norm_rope)
from .int8 import Int8RotLinear
from .kv_cache import CachePlan, cache_append, cached_attention
from .lowrank import fuse_qkv


def _frozen(t: Tensor) -> nn.Parameter:
    return nn.Parameter(t, requires_grad=False)


class AdapterBank(nn.Module):
    """The low-rank adapters of one projection, ``up[a] (down[a] x) * scale[a]`` for adapter a, as `adapter_add` takes
    them: ``down`` [adapters, rank, in], ``up`` [adapters, out, rank] (bfloat16), ``scale`` [adapters] (float32), frozen.
    The rank is rounded up to a multiple of 8; `load` fills one adapter of that rank or less (zero ranks add nothing)."""

    def __init__(self, in_features: int, out_features: int, adapters: int, rank: int) -> None:
        super().__init__()
        if adapters < 1 or rank < 1:
            raise ValueError(f"adapters and rank must be positive, got {adapters} and {rank}")
        self.in_features, self.out_features, self.adapters = in_features, out_features, adapters
        self.rank = -(-rank // 8) * 8
        self.down = _frozen(torch.zeros(adapters, self.rank, in_features, dtype=torch.bfloat16))
        self.up = _frozen(torch.zeros(adapters, out_features, self.rank, dtype=torch.bfloat16))
        self.scale = _frozen(torch.ones(adapters, dtype=torch.float32))

    def extra_repr(self) -> str:
        return f"{self.in_features} -> {self.out_features}, adapters={self.adapters}, rank={self.rank}"

    @torch.no_grad()
    def load(self, index: int, down: Tensor, up: Tensor, scale: float = 1.0) -> None:
        """Adapter ``index`` from ``down`` [r, in] and ``up`` [out, r], r up to the bank's rank."""
        if not 0 <= index < self.adapters:
            raise ValueError(f"adapter {index} of {self.adapters}")
        r = down.shape[0]
        if down.shape != (r, self.in_features) or up.shape != (self.out_features, r) or r > self.rank:
            raise ValueError(f"down must be [r, {self.in_features}] and up [{self.out_features}, r] with r up to "
                             f"{self.rank}, got {tuple(down.shape)} and {tuple(up.shape)}")
        self.down[index].zero_()
        self.up[index].zero_()
        self.down[index, :r] = down.to(self.down)
        self.up[index, :, :r] = up.to(self.up)
        self.scale[index] = scale

    def forward(self, y: Tensor, x: Tensor, plan: AdapterPlan, out: Tensor | None = None) -> Tensor:
        down, up, scale = self.down, self.up, self.scale
        if down.dtype is not y.dtype or scale.dtype is not torch.float32:  # after `Module.to`, as `Int8RotLinear`'s wscale
            down, up, scale = down.to(y.dtype), up.to(y.dtype), scale.to(torch.float32)
        return adapter_add(y, x, down, up, plan, scale=scale, out=out)


class AttentionBlock(nn.Module):
    """Multi-head attention whose projections are `Int8RotLinear`, over requests packed one behind the other.

    ``heads`` query heads share ``kv_heads`` key heads (default: as many); ``group`` is the Hadamard group of the
    projections, ``qk_norm`` gives queries and keys an RMS norm per head with weights, ``adapters`` and ``adapter_rank``
    an `AdapterBank` beside each projection. `from_projections` takes a model's own layers instead of empty ones."""

    def __init__(self, dim: int, heads: int, head_dim: int, group: int, *, kv_heads: int | None = None,
                 qk_norm: bool = True, eps: float = 1e-6, adapters: int = 0, adapter_rank: int = 0) -> None:
        super().__init__()
        kv_heads = heads if kv_heads is None else kv_heads
        self.dim, self.heads, self.kv_heads, self.head_dim, self.eps = dim, heads, kv_heads, head_dim, eps
        width = (heads + 2 * kv_heads) * head_dim
        self.qkv = Int8RotLinear(dim, width, group)
        self.out = Int8RotLinear(heads * head_dim, dim, group)
        self.norm_q = self.norm_k = None
        if qk_norm:
            self.norm_q = _frozen(torch.ones(head_dim, dtype=torch.bfloat16))
            self.norm_k = _frozen(torch.ones(head_dim, dtype=torch.bfloat16))
        self.qkv_adapters = self.out_adapters = None
        if adapters:
            self.qkv_adapters = AdapterBank(dim, width, adapters, adapter_rank)
            self.out_adapters = AdapterBank(heads * head_dim, dim, adapters, adapter_rank)

    @classmethod
    def from_projections(cls, to_q: Int8RotLinear, to_k: Int8RotLinear, to_v: Int8RotLinear, to_out: Int8RotLinear,
                         head_dim: int, *, norm_q: Tensor | None = None, norm_k: Tensor | None = None,
                         qk_norm: bool | None = None, **more) -> "AttentionBlock":
        """The block of a model's own projections: q, k and v fused into one layer (bitwise the same outputs).

        ``norm_q`` and ``norm_k`` are the weights [head_dim] of the model's RMS norms of query and key heads, kept in their
        type (their eps is ``eps``). Without them ``qk_norm`` says whether there are norms: False for a model that has
        none, True for norms whose weights are one, which is also taken, with a warning, when nothing is said."""
        if (norm_q is None) != (norm_k is None):
            raise ValueError("norm_q and norm_k come together")
        if norm_q is not None:
            if qk_norm is False:
                raise ValueError("qk_norm=False contradicts norm_q and norm_k")
            if norm_q.shape != (head_dim,) or norm_k.shape != (head_dim,):
                raise ValueError(f"norm_q and norm_k must be [{head_dim}], one weight a channel of a head, got "
                                 f"{tuple(norm_q.shape)} and {tuple(norm_k.shape)}")
        elif qk_norm is None:
            warnings.warn("from_projections without norm_q and norm_k: queries and keys get RMS norms whose weights are "
                          "one; give the model's weights, or qk_norm=False for none", UserWarning, stacklevel=2)
        if to_q.out_features % head_dim or to_k.out_features % head_dim or to_k.out_features != to_v.out_features:
            raise ValueError(f"projections of {to_q.out_features}, {to_k.out_features} and {to_v.out_features} columns "
                             f"are not heads of {head_dim}")
        if to_out.in_features != to_q.out_features:
            raise ValueError(f"to_out takes {to_out.in_features} columns, the heads give {to_q.out_features}")
        with torch.device("meta"):
            block = cls(to_q.in_features, to_q.out_features // head_dim, head_dim, to_q.group,
                        kv_heads=to_k.out_features // head_dim, qk_norm=qk_norm is not False, **more)
        device = to_q.qweight.device
        block.qkv, block.out = fuse_qkv(to_q, to_k, to_v), to_out
        for module in (block, block.qkv_adapters, block.out_adapters):
            for name, p in list(module._parameters.items()) if module is not None else ():
                if p is not None:
                    module._parameters[name] = _frozen((torch.zeros_like if name in ("down", "up") else torch.ones_like)(
                        p, device=device))
        if norm_q is not None:
            block.norm_q, block.norm_k = (_frozen(w.detach().to(device)) for w in (norm_q, norm_k))
        return block

    def forward(self, x: Tensor, plan: AttentionPlan | CachePlan, *, positions: Tensor | None = None,
                rotary: RotaryAxes | None = None, adapters: AdapterPlan | None = None, layer: int = 0) -> Tensor:
        """``x`` [tokens, dim] (bfloat16), the tokens of ``plan``'s sequences one behind the other; ``positions``
        [tokens, axes] with ``rotary``; ``adapters`` names the adapter of each request's tokens. With a `CachePlan` the
        tokens are the new ones of its requests: their keys and values are written to layer ``layer`` of its cache, and they
        attend to all that is held there. Forward only, as its operators are: x that requires a gradient is refused unless
        gradients are off."""
        if _differentiable():
            _forward_only("AttentionBlock", x)
        if adapters is not None and self.qkv_adapters is None:
            raise ValueError("the block was built without adapters")
        cached = isinstance(plan, CachePlan)
        if cached and plan.new_lengths != plan.q_lengths:
            raise ValueError("the block's tokens are both a step's queries and its new tokens")
        heads, kv_heads = self.heads, self.kv_heads
        qkv = self.qkv(x)
        if adapters is not None:
            self.qkv_adapters(qkv, x, adapters, out=qkv)
        parts = qkv.view(-1, heads + 2 * kv_heads, self.head_dim)
        q, k, v = parts[:, :heads], parts[:, heads:heads + kv_heads], parts[:, heads + kv_heads:]
        if self.norm_q is not None or rotary is not None:
            qk_norm_rope(q, k, positions, rotary, q_weight=self.norm_q, k_weight=self.norm_k,
                         norm=self.norm_q is not None, eps=self.eps, out=(q, k))
        if cached:
            cache_append(plan.cache, layer, k, v, plan)
            o = cached_attention(q, plan.cache, layer, plan)
        else:
            o = packed_attention(q, k, v, plan)
        o = o.view(-1, heads * self.head_dim)
        y = self.out(o)
        if adapters is not None:
            self.out_adapters(y, o, adapters, out=y)
        return y


__all__ = ["AdapterBank", "AttentionBlock"]

"""Transformer blocks whose linears are `Int8RotLinear`, over requests packed one behind the other: norms, modulation, gates
and residuals around an `AttentionBlock` and a feed-forward.

The reference's blocks do the same steps (src/hyperflow_h3_flash/transformer.py:339-380) one by one and for one request. Here
`residual_norm` takes what stands between two linears in one pass, across the end of a block too: a block's last residual and
the next block's first norm are one call (`TransformerStack`), unless the former's own norm has another eps than the latter."""

from __future__ import annotations

from collections.abc import Sequence

import torch
from torch import Tensor, nn

from .attention_block import AttentionBlock, _frozen
from .block import AdapterPlan, AttentionPlan, RotaryAxes, _differentiable, _forward_only
from .int8 import Int8RotLinear
from .kv_cache import CachePlan
from .residual_norm import NORMS, RowPlan, residual_norm


class TransformerBlock(nn.Module):
    """``x += gate * P(attention(N(x) * (1 + scale) + shift))``, then the same with the feed-forward ``down(up(.))``.

    ``up`` is an `Int8RotLinear` with the feed-forward's activation. N is ``norm`` ("rms" or "layer") and P ``post_norm`` (or
    None); ``weights`` gives each of them a weight [dim] (``norm_attention``, ``norm_ff``, ``post_attention``, ``post_ff``,
    ones at first, frozen)."""

    def __init__(self, attention: AttentionBlock, up: Int8RotLinear, down: Int8RotLinear, *, norm: str = "rms",
                 post_norm: str | None = None, weights: bool = True, eps: float = 1e-6) -> None:
        super().__init__()
        dim = attention.dim
        inner = up.out_features // (2 if (up.activation or "").startswith("swiglu") else 1)
        if up.in_features != dim or down.out_features != dim or down.in_features != inner:
            raise ValueError(f"the feed-forward takes {up.in_features} columns to {inner} and {down.in_features} to "
                             f"{down.out_features}, the attention block has {dim}")
        if norm not in NORMS or norm is None or post_norm not in NORMS:
            raise ValueError(f"a norm is one of {tuple(NORMS)}, and not None before a branch, got {norm!r} and {post_norm!r}")
        self.dim, self.norm, self.post_norm, self.eps = dim, norm, post_norm, eps
        self.attention, self.up, self.down = attention, up, down
        device = up.qweight.device
        for name, there in (("norm_attention", weights), ("norm_ff", weights), ("post_attention", weights and post_norm),
                            ("post_ff", weights and post_norm)):
            setattr(self, name, _frozen(torch.ones(dim, dtype=torch.bfloat16, device=device)) if there else None)

    def forward(self, x: Tensor, plan: AttentionPlan | CachePlan, *, modulation: Tensor | None = None,
                rows: RowPlan | None = None, positions: Tensor | None = None, rotary: RotaryAxes | None = None,
                adapters: AdapterPlan | None = None, layer: int = 0) -> Tensor:
        """``x`` [tokens, dim], the residual stream (bfloat16 or float32). ``modulation`` [requests, 6, dim] with ``rows``, or
        [1, 6, dim] for all tokens: shift, scale and gate of the attention, then of the feed-forward. The other arguments are
        `AttentionBlock`'s."""
        return _run([self], x, plan, None if modulation is None else [modulation], rows, positions, rotary, adapters, layer)


class TransformerStack(nn.Module):
    """Blocks one behind the other; with a `CachePlan`, block i keeps its keys and values in layer i of the cache."""

    def __init__(self, blocks: Sequence[TransformerBlock]) -> None:
        super().__init__()
        self.blocks = nn.ModuleList(blocks)
        if any(b.dim != self.blocks[0].dim for b in self.blocks):
            raise ValueError(f"blocks of different widths: {sorted({b.dim for b in self.blocks})}")

    def forward(self, x: Tensor, plan: AttentionPlan | CachePlan, *, modulation: Sequence[Tensor] | None = None,
                rows: RowPlan | None = None, positions: Tensor | None = None, rotary: RotaryAxes | None = None,
                adapters: AdapterPlan | None = None) -> Tensor:
        """As `TransformerBlock`'s, with a ``modulation`` for each block."""
        return _run(list(self.blocks), x, plan, modulation, rows, positions, rotary, adapters, 0)


def _run(blocks: list[TransformerBlock], x: Tensor, plan, modulation: Sequence[Tensor] | None, rows: RowPlan | None,
         positions, rotary, adapters, layer: int) -> Tensor:
    if _differentiable():
        _forward_only("TransformerBlock", x, *(modulation or ()))
    if modulation is not None and len(modulation) != len(blocks):
        raise ValueError(f"{len(modulation)} modulations for {len(blocks)} blocks")
    for m in modulation or ():
        if m.dim() != 3 or m.shape[1:] != (6, blocks[0].dim):
            raise ValueError(f"a modulation must be [requests, 6, {blocks[0].dim}], got {tuple(m.shape)}")
    if not blocks:
        return x
    kind = torch.float16 if x.dtype is torch.float16 else torch.bfloat16

    def weight(w: Tensor | None) -> Tensor | None:  # after `Module.to`, as `AdapterBank`'s
        return w if w is None or w.dtype is kind or w.dtype is torch.float32 else w.to(torch.float32)

    of = [(None,) * 6 if modulation is None else modulation[i].unbind(1) for i in range(len(blocks))]
    shift, scale = of[0][:2]
    _, n = residual_norm(x, rows=rows, norm=blocks[0].norm, weight=weight(blocks[0].norm_attention), scale=scale, shift=shift,
                         eps=blocks[0].eps)
    for i, block in enumerate(blocks):
        gate, ff_shift, ff_scale, ff_gate = of[i][2:]
        a = block.attention(n, plan, positions=positions, rotary=rotary, adapters=adapters, layer=layer + i)
        x, n = residual_norm(x, a, rows=rows, gate=gate, post_norm=block.post_norm, post_weight=weight(block.post_attention),
                             norm=block.norm, weight=weight(block.norm_ff), scale=ff_scale, shift=ff_shift, eps=block.eps)
        f = block.down(block.up(n))
        after = blocks[i + 1] if i + 1 < len(blocks) else None
        shift, scale = of[i + 1][:2] if after is not None else (None, None)
        if after is not None and block.post_norm is not None and block.eps != after.eps:  # an eps each: two calls
            x, _ = residual_norm(x, f, rows=rows, gate=ff_gate, post_norm=block.post_norm, post_weight=weight(block.post_ff),
                                 norm=None, eps=block.eps)
            _, n = residual_norm(x, rows=rows, norm=after.norm, weight=weight(after.norm_attention), scale=scale, shift=shift,
                                 eps=after.eps)
            continue
        x, n = residual_norm(x, f, rows=rows, gate=ff_gate, post_norm=block.post_norm, post_weight=weight(block.post_ff),
                             norm=None if after is None else after.norm,
                             weight=None if after is None else weight(after.norm_attention), scale=scale, shift=shift,
                             eps=block.eps if after is None else after.eps)
    return x


__all__ = ["TransformerBlock", "TransformerStack"]

"""The 4-bit cache's operators (``kv_cache.py``) and the residual norms (``residual_norm.py``) on host tensors: the kernels'
definitions in float64, rounded once, and the same bytes in the pages."""

from __future__ import annotations

from collections.abc import Sequence
from types import SimpleNamespace

import torch
from torch import Tensor

from . import host_block

#: Channels that share a scale.
GROUP = 32
LEVELS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
#: Borders between neighbouring levels, and whether the border itself goes down (to the even code).
BORDERS = ((0.25, True), (0.75, False), (1.25, True), (1.75, False), (2.5, True), (3.5, False), (5.0, True))
#: Least and largest exponent of a scale.
EXPONENTS = {torch.bfloat16: (-125, 125), torch.float16: (-23, 13)}
NAN_SCALE = 255


def scale_bytes(groups: int) -> int:
    return 4 if groups == 3 else groups


def slab_bytes(groups: int, page_size: int) -> int:
    """Bytes of a page's tokens of one head."""
    return page_size * 2 * (16 * groups + scale_bytes(groups))


def quantize(x: Tensor) -> tuple[Tensor, Tensor]:
    """``x`` [..., D] as (packed codes uint8 [..., groups, 16], scale bytes uint8 [..., groups])."""
    groups = -(-x.shape[-1] // GROUP)
    h = torch.nn.functional.pad(x.double(), (0, groups * GROUP - x.shape[-1])).unflatten(-1, (groups, GROUP))
    finite = h.isfinite().all(-1)
    h = torch.where(finite[..., None], h, 0.0)
    m, e = torch.frexp(h.abs().amax(-1))
    e = (e - torch.where(m <= 0.875, 3, 2)).clamp(*EXPONENTS[x.dtype])
    a = torch.ldexp(h.abs(), -e[..., None])
    code = torch.zeros(a.shape, dtype=torch.uint8)
    for border, down in BORDERS:
        code += (a > border) if down else (a >= border)
    code |= torch.signbit(h).to(torch.uint8) << 3
    return code[..., 0::2] | (code[..., 1::2] << 4), torch.where(finite, e + 127, NAN_SCALE).to(torch.uint8)


def dequantize(codes: Tensor, scales: Tensor, dim: int, dtype: torch.dtype) -> Tensor:
    levels = torch.cat([LEVELS, -LEVELS])
    h = levels[torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2).long()]
    h = torch.ldexp(h, scales[..., None].int() - 127)
    h = torch.where((scales == NAN_SCALE)[..., None], torch.nan, h)
    return h.flatten(-2)[..., :dim].to(dtype)


def _views(cache, layer: int) -> tuple[Tensor, Tensor]:
    """A layer's pages as codes [pages, heads, k or v, groups, page_size, 16] and scales [pages, heads, page_size, k or v,
    bytes]."""
    G, P, S = cache.groups, cache.page_size, scale_bytes(cache.groups)
    slabs = cache.data[layer].view(cache.pages, cache.kv_heads, -1)
    return (slabs[..., :2 * G * P * 16].unflatten(-1, (2, G, P, 16)), slabs[..., 2 * G * P * 16:].unflatten(-1, (P, 2, S)))


def _slots(cache, table: Sequence[int], first: int, last: int) -> tuple[Tensor, Tensor]:
    """(page, place in it) of a request's tokens first .. last - 1."""
    at = torch.arange(first, last)
    return torch.tensor(list(table), dtype=torch.int64)[at // cache.page_size], at % cache.page_size


def append(cache, layer: int, k: Tensor, v: Tensor, plan) -> None:
    codes, scales = _views(cache, layer)
    G, row = cache.groups, 0
    for table, total, new in zip(plan.tables, plan.kv_lengths, plan.new_lengths):
        page, at = _slots(cache, table, total - new, total)
        for which, x in enumerate((k, v)):
            c, s = quantize(x[row:row + new])
            codes[page, :, which, :, at] = c
            scales[page, :, at, which, :G] = s
        row += new


def read(cache, layer: int, plan, k: Tensor, v: Tensor) -> None:
    codes, scales = _views(cache, layer)
    G, row = cache.groups, 0
    for table, total in zip(plan.tables, plan.kv_lengths):
        page, at = _slots(cache, table, 0, total)
        for which, x in enumerate((k, v)):
            x[row:row + total] = dequantize(codes[page, :, which, :, at], scales[page, :, at, which, :G], cache.head_dim,
                                            cache.dtype)
        row += total


def attention(q: Tensor, cache, layer: int, plan, scale: float) -> Tensor:
    k, v = (torch.empty(plan._kv_shape, dtype=cache.dtype) for _ in range(2))
    read(cache, layer, plan, k, v)
    packed = SimpleNamespace(heads=plan.heads, kv_heads=plan.kv_heads, q_lengths=plan.q_lengths, kv_lengths=plan.kv_lengths,
                             causal=plan.causal)
    return host_block.packed_attention(q, k, v, packed, scale)


def _normed(h: Tensor, kind: str | None, weight: Tensor | None, eps: float) -> Tensor:
    if kind == "layer":
        h = h - h.mean(-1, keepdim=True)
    if kind is not None:
        h = h / torch.sqrt(h.square().mean(-1, keepdim=True) + eps)
    return h if weight is None else h * weight.double()


def residual_norm(x, y, rows, residual, gate, post_norm, post_weight, norm, weight, scale, shift, eps, dtype, want):
    def of_rows(t: Tensor) -> Tensor:
        t = t.double()
        return t if t.dim() == 1 or t.shape[0] == 1 or rows is None else t[rows.groups.long()]

    h = x.double()
    r = x
    if y is not None:
        branch = _normed(y.double(), post_norm, post_weight, eps)
        h = residual * h + (branch if gate is None else of_rows(gate) * branch)
        r = h.to(x.dtype)
    if not want:
        return r, None
    h = _normed(h, norm, weight, eps)
    if scale is not None:
        h = h * (1 + of_rows(scale))
    if shift is not None:
        h = h + of_rows(shift)
    return r, h.to(dtype)

"""The attention block's operators (``block.py``) on host tensors: the kernels' definitions in float64, rounded once to
the inputs' type."""

from __future__ import annotations

import torch
from torch import Tensor


def _rotate(x: Tensor, weight: Tensor | None, phase: Tensor | None, interleaved: bool, norm: bool, eps: float) -> Tensor:
    h = x.double()
    if norm:
        h = h / torch.sqrt(h.square().mean(-1, keepdim=True) + eps)
        if weight is not None:
            h = h * weight.double()
    if phase is not None:
        pairs = phase.shape[-1]
        cos, sin = phase.cos()[:, None], phase.sin()[:, None]
        a, b = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if interleaved else (slice(0, pairs),
                                                                                    slice(pairs, 2 * pairs))
        turned = h.clone()
        turned[..., a] = h[..., a] * cos - h[..., b] * sin
        turned[..., b] = h[..., a] * sin + h[..., b] * cos
        h = turned
    return h.to(x.dtype)


def qk_norm_rope(q, k, positions, rotary, q_weight, k_weight, norm, eps):
    phase, interleaved = None, False
    if rotary is not None:
        phase = positions.double()[:, rotary.axis.long()] * rotary.rates
        interleaved = rotary.interleaved
    return (_rotate(q, q_weight, phase, interleaved, norm, eps),
            None if k is None else _rotate(k, k_weight, phase, interleaved, norm, eps))


def packed_attention(q: Tensor, k: Tensor, v: Tensor, plan, scale: float) -> Tensor:
    out = torch.zeros(q.shape, dtype=q.dtype)
    group = plan.heads // plan.kv_heads
    q0 = k0 = 0
    for nq, nk in zip(plan.q_lengths, plan.kv_lengths):
        first = max(nq - nk, 0) if plan.causal else 0 if nk else nq  # queries before it see no key
        qs = q[q0 + first:q0 + nq].double()
        ks, vs = k[k0:k0 + nk].double(), v[k0:k0 + nk].double()
        for h in range(plan.heads):
            for i in range(0, nq - first, 512):
                rows = qs[i:i + 512, h]
                s = (rows @ ks[:, h // group].t()) * scale
                sees = torch.ones_like(s, dtype=torch.bool)
                if plan.causal:
                    sees = sees.tril(first + i + nk - nq)
                w = torch.softmax(s.masked_fill(~sees, -torch.inf), dim=-1)
                values = vs[:, h // group]
                o = w @ values.nan_to_num(0.0, 0.0, 0.0)
                for j in torch.nonzero(~values.isfinite().all(-1))[:, 0].tolist():  # added only where they are seen
                    odd = torch.where(values[j].isfinite(), 0.0, values[j])
                    o += torch.where(sees[:, j:j + 1], odd, 0.0)
                out[q0 + first + i:q0 + first + i + len(rows), h] = o.to(q.dtype)
        q0, k0 = q0 + nq, k0 + nk
    return out


def adapter_add(y: Tensor, x: Tensor, down: Tensor, up: Tensor, plan, scale: Tensor | None) -> Tensor:
    out = y.clone()
    rows = torch.repeat_interleave(torch.tensor(plan.ids, dtype=torch.int64), torch.tensor(plan.lengths,
                                                                                          dtype=torch.int64))
    for a in sorted(set(plan.ids)):
        at = torch.nonzero(rows == a)[:, 0]
        if a < 0 or not len(at):
            continue
        delta = (x[at].double() @ down[a].double().t()) @ up[a].double().t()
        out[at] = (y[at].double() + (1.0 if scale is None else scale[a].double()) * delta).to(y.dtype)
    return out

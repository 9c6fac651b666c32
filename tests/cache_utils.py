"""Plain 64-bit forms of the 4-bit cache and of the residual norms, and the error bounds their tests hold results to.

What is read from a cache has one right value: a nearest level (ties to the even code) times a power of two, exact in either
type. Attention over it has the bound of packed attention (block_utils.py) on those values."""

from __future__ import annotations

import math

import torch

import block_utils as U

LEVELS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
LIMITS = {torch.bfloat16: (-125, 125), torch.float16: (-23, 13)}
UNIT = {**U.UNIT, torch.float32: 2.0 ** -24}
TINY = {**U.TINY, torch.float32: 2.0 ** -150}


def held(x):
    """The values (float64) that x [..., D] is read as: the nearest of the levels by distance, the even one of two as near."""
    low, high = LIMITS[x.dtype]
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for c in range(0, x.shape[-1], 32):
        h = x[..., c:c + 32].double()
        finite = h.isfinite().all(-1, keepdim=True)
        top = torch.where(finite, h, 0.0).abs().amax(-1, keepdim=True)
        e = torch.full_like(top, low)
        for i in range(low, high):  # the least power of two that is a seventh of the largest
            e = torch.where(top > 7 * 2.0 ** i, i + 1.0, e)
        s = torch.exp2(e)
        off = (h.abs()[..., None] / s[..., None] - torch.tensor(LEVELS, dtype=torch.float64, device=x.device)).abs()
        off = off + 1e-9 * (torch.arange(8, device=x.device) % 2)  # of two as near the even code (quotients have 11 bits)
        value = torch.tensor(LEVELS, dtype=torch.float64, device=x.device)[off.argmin(-1)] * s
        out[..., c:c + 32] = torch.where(finite, torch.where(h < 0, -value, value), math.nan)
    return out


def attention(q, k, v, q_lens, kv_lens, causal, scale):
    """(result, bound) of attention over what is held of k and v."""
    return U.attention(q, held(k).to(k.dtype), held(v).to(v.dtype), q_lens, kv_lens, causal, scale)


# The kernel's sums over a row: up to 32 terms a lane, 6 exchanges and up to 8 waves are 46 additions one behind the other;
# with the products' own roundings fewer than 64 roundings of the terms' magnitudes.
SUM = 64 * 2.0 ** -24


def normed(h, e, kind, weight, eps):
    """(norm of h, error bound) for h known up to e."""
    if kind is not None:
        if kind == "layer":
            mean = h.mean(-1, keepdim=True)
            off = e.mean(-1, keepdim=True) + SUM * h.abs().mean(-1, keepdim=True)
            h = h - mean
            e = e + off + 2.0 ** -24 * h.abs()
        var = h.pow(2).mean(-1, keepdim=True)
        dvar = 2 * (h.abs() * e).mean(-1, keepdim=True) + e.pow(2).mean(-1, keepdim=True) + SUM * var
        sigma = torch.sqrt(var + eps)
        h, e = h / sigma, e / sigma
        # The root's relative error is half the sum's (all of it here), then the eps, sum, root, quotient and product round.
        e = e + h.abs() * (dvar / (var + eps) + 8 * 2.0 ** -24)
    if weight is not None:
        w = weight.double()
        h, e = h * w, e * w.abs() + 2.0 ** -24 * (h * w).abs()
    return h, e


def residual_norm(x, y, groups, residual, gate, post, post_weight, norm, weight, scale, shift, eps, dtype):
    """((r, bound), (n, bound)); ``groups``: the row of gate, scale and shift for each row (None: they have one)."""
    def rows(t):
        t = t.double()
        return t if t.dim() == 1 or groups is None else t[groups]

    u = 2.0 ** -24
    h, e = x.double(), torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    r = None
    if y is not None:
        b, be = normed(y.double(), torch.zeros_like(e), post, post_weight, eps)
        if gate is not None:
            b, be = b * rows(gate), be * rows(gate).abs() + u * (b * rows(gate)).abs()
        f = torch.tensor(residual, dtype=torch.float32).double().item()
        h = f * h + b
        e = be + u * h.abs()
        r = (h, UNIT[x.dtype] * (h.abs() + e) + e + TINY[x.dtype])
    n, ne = normed(h, e, norm, weight, eps)
    if scale is not None:
        f = 1 + rows(scale)
        n, ne = n * f, ne * f.abs() + 2 * u * (n * f).abs() + u * n.abs()
    if shift is not None:
        n = n + rows(shift)
        ne = ne + u * n.abs()
    return r, (n, UNIT[dtype] * (n.abs() + ne) + ne + TINY[dtype])

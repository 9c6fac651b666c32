"""Plain 64-bit forms of the attention block's operators and the error bounds their tests hold the results to.

The bounds follow from the types. Rounding a result once to a type of p significant bits errs by at most u |result|,
u = 2^-p (p is 8 for bfloat16, 11 for float16), plus half the smallest step of the type. Sums in float32 of n products err by at
most n 2^-24 times the sum of the products' magnitudes."""

from __future__ import annotations

import torch

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
#: Half the distance of the type's smallest values.
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}


def rotate(x, weight, positions, dims, theta, interleaved, norm, eps=1e-6):
    """(result, bound) in float64 of one tensor [T, H, D]; dims None: no rotation."""
    h = x.double()
    D = h.shape[-1]
    if norm:
        h = h * (h.pow(2).sum(-1, keepdim=True) / D + eps).rsqrt()
        if weight is not None:
            h = h * weight.double()
    size = h.abs()
    if dims is not None:
        angles = torch.cat([positions[:, a].double()[:, None] * theta ** (-torch.arange(0, n, 2, dtype=torch.float64,
                                                                                      device=x.device) / n)
                            for a, n in enumerate(dims)], dim=-1)[:, None, :]
        P = angles.shape[-1]
        if interleaved:
            first, second = list(range(0, 2 * P, 2)), list(range(1, 2 * P, 2))
        else:
            first, second = list(range(P)), list(range(P, 2 * P))
        a, b = h[..., first], h[..., second]
        r = h.clone()
        r[..., first] = a * angles.cos() - b * angles.sin()
        r[..., second] = b * angles.cos() + a * angles.sin()
        both = a.abs() + b.abs()
        size = size.clone()
        size[..., first] = both
        size[..., second] = both
        h = r
    # The norm's sum of D squares, its square root and quotient, the weight, sine and cosine (2 units in the last place
    # each) and two products: fewer than (D / 2 + 32) roundings of the pair's magnitude.
    return h, UNIT[x.dtype] * h.abs() + (D / 2 + 32) * 2.0 ** -24 * size + TINY[x.dtype]


def attention(q, k, v, q_lens, kv_lens, causal, scale):
    """(result, bound) in float64 of packed attention; a row without a key is zero, with bound zero."""
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    group = q.shape[1] // k.shape[1]
    D = q.shape[2]
    u, tiny = UNIT[q.dtype], TINY[q.dtype]
    q0 = k0 = 0
    for nq, nk in zip(q_lens, kv_lens):
        for h in range(q.shape[1] if nq and nk else 0):
            a, b, w = q[q0:q0 + nq, h].double(), k[k0:k0 + nk, h // group].double(), v[k0:k0 + nk, h // group].double()
            s = a @ b.t().contiguous() * scale
            rough = a.abs() @ b.abs().t().contiguous() * scale
            sees = torch.ones(nq, nk, dtype=torch.bool, device=q.device)
            if causal:
                sees = torch.arange(nk, device=q.device)[None] <= torch.arange(nq, device=q.device)[:, None] + nk - nq
            any_key = sees.any(-1, keepdim=True)
            p = torch.softmax(torch.where(sees, s, -torch.inf), -1)
            p = torch.where(any_key, p, 0.0)
            o = p @ w
            size = p @ w.abs()
            # A score errs by D / 2 float32 roundings of its products on average and D at most, which moves a weight by
            # that much in proportion; the weight is rounded to the type, and sums run over nk keys.
            off = (torch.where(sees, rough, 0.0).amax(-1, keepdim=True) * 2 * (D + 4) + nk) * 2.0 ** -24
            out[q0:q0 + nq, h] = o
            bound[q0:q0 + nq, h] = torch.where(
                any_key, u * o.abs() + (u + off) * size + tiny * (1 + nk * w.abs().max()), 0.0)
        q0, k0 = q0 + nq, k0 + nk
    return out, bound


def adapters(y, x, down, up, ids, lens, scale):
    out = y.double().clone()
    slack = torch.zeros_like(out)
    m = 0
    for a, n in zip(ids, lens):
        if a >= 0 and n:
            f = 1.0 if scale is None else scale[a].double()
            A, B = down[a].double().t().contiguous(), up[a].double().t().contiguous()
            out[m:m + n] += f * ((x[m:m + n].double() @ A) @ B)
            slack[m:m + n] = f * ((x[m:m + n].double().abs() @ A.abs()) @ B.abs())
        m += n
    # The sums of K and r products in float32, and the intermediate kept to two 8-bit (bfloat16) mantissas.
    K, r = x.shape[1], down.shape[1]
    return out, UNIT[y.dtype] * out.abs() + (2.0 ** -16 + (K + 2 * r + 8) * 2.0 ** -24) * slack + TINY[y.dtype]


def check(got, ref, bound, what=""):
    got = got.double()
    assert got.shape == ref.shape
    nan = ref.isnan()
    assert torch.equal(got.isnan(), nan), f"{what}: NaN in other places"
    off = torch.where(nan | (got == ref), 0.0, (got - ref).abs())
    bad = off > bound * (1 + 1e-12)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / bound.clamp_min(1e-300)).max()):.3g} bounds"

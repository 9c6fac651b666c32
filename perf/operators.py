"""The performance cases of the attention block's operators around the INT8 linears: the per-head norms of queries and
keys with the rotation of positions on several axes, attention over packed sequences, and low-rank adapters of many
requests beside a shared projection.

A case names one call (``op``) and its sizes:

* ``qk_norm_rope``: q [T, Hq, D] and k [T, Hk, D] as views of one fused projection's output [T, (Hq + 2 Hk) D].
* ``attention``: packed sequences; ``q_lens`` and ``kv_lens`` are texts of comma-separated lengths.
* ``adapters``: rows [M, K] of several requests, each with an adapter or none, added to a projection's output [M, N].

``run`` computes them in plain fp32 torch operations, or with ``own`` set through this framework's entry points.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
#: The most multiply-adds x 2 of a listed attention case (one GPU's heads of a whole clip); a drawn case stays below.
MOST_FLOPS = 4.0 * 37710 * 37710 * 7 * 128
#: The most bytes of a listed case of the other two operators; a drawn case stays below.
MOST_BYTES = 2.2e9


def _ints(text):
    return [int(v) for v in text.split(",")]


def _text(values):
    return ",".join(str(v) for v in values)


def _rope(name, T, hq, hk, D, axes, theta, interleaved, norm, dtype="bf16"):
    return {"name": name, "op": "qk_norm_rope", "T": T, "hq": hq, "hk": hk, "D": D, "axes": axes, "theta": theta,
            "interleaved": interleaved, "norm": norm, "dtype": dtype}


def _attention(name, q_lens, kv_lens, hq, hk, D, causal, dtype="bf16"):
    return {"name": name, "op": "attention", "q_lens": q_lens, "kv_lens": kv_lens, "hq": hq, "hk": hk, "D": D,
            "causal": causal, "dtype": dtype}


def _adapters(name, lens, ids, adapters, rank, K, N, dtype="bf16"):
    return {"name": name, "op": "adapters", "lens": lens, "ids": ids, "adapters": adapters, "rank": rank, "K": K,
            "N": N, "dtype": dtype}


def listed():
    return [
        # The model's 5.2 s clip: 37710 video tokens, 56 heads of 128, time, height and width on 44 + 42 + 42 channels.
        _rope("rope_clip", 37710, 56, 56, 128, "44,42,42", 10000.0, True, True),
        # A packed batch of prompts through a grouped-head text encoder: one axis, halves rotated, no norm.
        _rope("rope_prompts", 4099, 32, 8, 128, "128", 1000000.0, False, False, "fp16"),
        # One new token of each of a few requests: launch latency.
        _rope("rope_rows", 7, 32, 8, 128, "32,48,48", 10000.0, False, True),
        # One GPU's heads of the clip under an 8-way head split: every token against every token.
        _attention("attn_clip", "37710", "37710", 7, 7, 128, False),
        # Clips and images of several requests packed in one batch, all heads.
        _attention("attn_packed", "5168,1001,2600,77", "5168,1001,2600,77", 56, 56, 128, False),
        # Prompts of a text encoder: causal, grouped heads, ragged lengths.
        _attention("attn_prompts", "4099,1537,300,61,2048", "4099,1537,300,61,2048", 32, 8, 128, True),
        # Video tokens against the text tokens of their own request: cross attention, few keys.
        _attention("attn_cross", "5168,2600", "511,77", 56, 56, 128, False),
        # Serving: one new token of each request against its own cache.
        _attention("attn_tokens", _text([1] * 16), _text([8191, 4096, 733, 1, 16384, 2500, 6001, 127, 9999, 3000, 512,
                                                          7777, 64, 12001, 1025, 5000]), 32, 8, 128, True),
        # One short prompt of a small encoder: the smallest call.
        _attention("attn_short", "77", "77", 12, 12, 64, True, "fp16"),
        # Sixteen adapters over 64 single rows of as many requests, some without an adapter.
        _adapters("adapters_rows", _text([1] * 64), _text([(i * 7) % 17 - 1 for i in range(64)]), 16, 16, 5120, 5120),
        # A packed batch of images, ragged, one request without an adapter.
        _adapters("adapters_packed", "1001,77,2600,300,64", "2,0,1,-1,2", 3, 64, 5376, 7168),
        # A whole clip's tokens of two requests beside the fused q/k/v projection: the largest.
        _adapters("adapters_clip", "20000,12768", "1,0", 2, 32, 5120, 15360),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["qk_norm_rope", "attention", "attention", "adapters"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    while True:
        if op == "qk_norm_rope":
            D = rng.choice([64, 96, 128, 128])
            hk = rng.choice([1, 2, 7, 8, 12, 56])
            hq = hk * rng.choice([1, 1, 3, 4, 8])
            axes = {64: ["64", "16,24,24"], 96: ["96", "32,32,32", "32,32"], 128: ["128", "44,42,42", "32,48,48", "64"]}
            case = _rope("", _log_int(rng, 1, 40000), hq, hk, D, rng.choice(axes[D]), rng.choice([1e4, 1e6]),
                         rng.random() < 0.5, rng.random() < 0.7, dtype)
            fits = work(case)["bytes"] <= MOST_BYTES
        elif op == "attention":
            D = rng.choice([64, 80, 96, 128, 128, 128])
            hk = rng.choice([1, 2, 4, 7, 8, 12])
            hq = hk * rng.choice([1, 1, 2, 4, 5, 8])
            count = _log_int(rng, 1, 24)
            longest = _log_int(rng, 16, 24000)
            kv = [max(1, min(longest, _log_int(rng, max(1, longest // 16), longest))) for _ in range(count)]
            form = rng.choice(["self", "self", "self", "tokens", "cross", "tail"])
            if form == "self":
                q = kv
            elif form == "tokens":
                q = [1] * count
            elif form == "cross":
                q = [_log_int(rng, 16, 6000) for _ in range(count)]
            else:  # a prompt's last part against all that is cached
                q = [_log_int(rng, 1, v) for v in kv]
            causal = form != "cross" and rng.random() < 0.6
            case = _attention("", _text(q), _text(kv), hq, hk, D, causal, dtype)
            fits = sum(4.0 * D * hq * a * b for a, b in zip(q, kv)) <= MOST_FLOPS and work(case)["bytes"] <= MOST_BYTES
        else:
            count = _log_int(rng, 1, 64)
            longest = _log_int(rng, 1, 30000 // count)
            lens = [_log_int(rng, max(1, longest // 8), longest) for _ in range(count)]
            adapters = rng.randint(1, 16)
            ids = [rng.randint(-1, adapters - 1) for _ in range(count)]
            case = _adapters("", _text(lens), _text(ids), adapters, 8 * rng.randint(1, 16), 256 * rng.randint(4, 56),
                             8 * _log_int(rng, 128, 2688), dtype)
            fits = work(case)["bytes"] <= MOST_BYTES and 3072 not in (case["K"], case["N"])
        if fits:
            del case["name"]
            return case


def work(case):
    if case["op"] == "qk_norm_rope":
        n = case["T"] * (case["hq"] + case["hk"]) * case["D"]
        return {"bytes": 4 * n + 4 * case["T"] * len(_ints(case["axes"])), "flops": (9 if case["norm"] else 3) * n}
    if case["op"] == "attention":
        q, kv, D = _ints(case["q_lens"]), _ints(case["kv_lens"]), case["D"]
        if case["causal"]:  # row i of a sequence sees i + 1 + (kv - q) keys
            pairs = sum(sum(min(max(i + 1 + b - a, 0), b) for i in range(a)) for a, b in zip(q, kv))
        else:
            pairs = sum(a * b for a, b in zip(q, kv))
        return {"bytes": 4 * D * (sum(q) * case["hq"] + sum(kv) * case["hk"]), "flops": 4 * D * case["hq"] * pairs}
    lens, ids = _ints(case["lens"]), _ints(case["ids"])
    K, N, r = case["K"], case["N"], case["rank"]
    rows = sum(n for n, a in zip(lens, ids) if a >= 0)
    used = len({a for a in ids if a >= 0})
    return {"bytes": 2 * (rows * K + 2 * sum(lens) * N + used * r * (K + N)), "flops": 2 * rows * r * (K + N)}


# ------------------------------------------------------------------------------------------------------------- inputs

def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _inputs(case, seed):
    """The inputs of a case, from the seed alone, as tensors and plain values."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "qk_norm_rope":
        T, hq, hk, D = case["T"], case["hq"], case["hk"], case["D"]
        # A fused projection's output: some channels stronger than others, as a transformer's are.
        gain = torch.exp(0.5 * _normal(gen, (hq + 2 * hk) * D))
        qkv = (_normal(gen, T, (hq + 2 * hk) * D) * gain).to(dtype)
        axes = _ints(case["axes"])
        # Positions of a grid walked row by row (time slowest), behind a prompt; one axis counts the tokens.
        at = torch.arange(T, device="cuda") + seed % 5
        positions = at[:, None] if len(axes) == 1 else torch.stack(
            [at // 1620] + [(at // 54) % 30, at % 54][:len(axes) - 1], dim=1)
        weights = ((1 + 0.2 * _normal(gen, 2, D)).to(dtype)) if case["norm"] else None
        return {"q": qkv[:, :hq * D].view(T, hq, D), "k": qkv[:, hq * D:(hq + hk) * D].view(T, hk, D),
                "positions": positions.to(torch.int32).contiguous(), "weights": weights}
    if case["op"] == "attention":
        q_lens, kv_lens = _ints(case["q_lens"]), _ints(case["kv_lens"])
        hq, hk, D = case["hq"], case["hk"], case["D"]
        # Normed queries and keys (scores of a few units either way), values with a mean of their own per channel; the
        # values are a view of the fused projection's output where queries and keys come from the same tokens.
        q = (1.5 * _normal(gen, sum(q_lens), hq, D)).to(dtype)
        k = (1.3 * _normal(gen, sum(kv_lens), hk, D)).to(dtype)
        v = _normal(gen, sum(kv_lens), hk, D) + 0.5 * _normal(gen, hk, D)
        if q_lens == kv_lens:
            wide = torch.zeros(sum(kv_lens), hq + 2 * hk, D, device="cuda", dtype=dtype)
            wide[:, hq + hk:] = v
            v = wide[:, hq + hk:]
        else:
            v = v.to(dtype)
        return {"q": q, "k": k, "v": v, "q_lens": q_lens, "kv_lens": kv_lens}
    lens, ids = _ints(case["lens"]), _ints(case["ids"])
    M, K, N, r = sum(lens), case["K"], case["N"], case["rank"]
    x = _normal(gen, M, K)
    x[:, ::199] *= 10  # outlier channels, as the INT8 layers' inputs have
    return {"x": x.to(dtype), "y": _normal(gen, M, N).to(dtype), "lens": lens, "ids": ids,
            "down": (_normal(gen, case["adapters"], r, K) / math.sqrt(K)).to(dtype),
            "up": (_normal(gen, case["adapters"], N, r) / math.sqrt(r)).to(dtype),
            "scale": 0.25 + 0.5 * torch.rand(case["adapters"], generator=gen, device="cuda")}


def prepare(case, seed):
    state = {"case": case, **_inputs(case, seed)}
    if own:
        import hyperflow_h3_flash_amd as hf

        if case["op"] == "qk_norm_rope":
            state["rotary"] = hf.RotaryAxes(_ints(case["axes"]), theta=case["theta"], interleaved=case["interleaved"])
        elif case["op"] == "attention":
            state["plan"] = hf.AttentionPlan(state["q_lens"], state["kv_lens"], heads=case["hq"], kv_heads=case["hk"],
                                             head_dim=case["D"], causal=case["causal"], device="cuda")
        else:
            state["plan"] = hf.AdapterPlan(state["ids"], state["lens"], adapters=case["adapters"], device="cuda")
    elif case["op"] == "adapters":  # the plain form's plan: which rows belong to each adapter
        rows = torch.repeat_interleave(torch.tensor(state["ids"]), torch.tensor(state["lens"]))
        state["rows"] = [(a, torch.nonzero(rows == a)[:, 0].cuda()) for a in sorted(set(state["ids"])) if a >= 0]
    return state


# --------------------------------------------------------------------------------------------------- the plain forms

def _plain_rotate(x, weight, cos, sin, interleaved, norm):
    h = x.float()
    if norm:
        h = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-6) * weight.float()
    R = 2 * cos.shape[-1]
    turn, rest = h[..., :R], h[..., R:]
    if interleaved:
        a, b = turn[..., 0::2], turn[..., 1::2]
        turn = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
    else:
        a, b = turn[..., :R // 2], turn[..., R // 2:]
        turn = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
    return torch.cat([turn, rest], dim=-1).to(x.dtype)


def _plain_qk_norm_rope(state):
    case, positions = state["case"], state["positions"]
    angles = []
    for axis, dim in enumerate(_ints(case["axes"])):
        rates = case["theta"] ** (-torch.arange(0, dim, 2, device="cuda", dtype=torch.float32) / dim)
        angles.append(positions[:, axis:axis + 1].float() * rates)
    angles = torch.cat(angles, dim=-1)[:, None, :]
    cos, sin = angles.cos(), angles.sin()
    w = state["weights"]
    return tuple(_plain_rotate(state[name], None if w is None else w[i], cos, sin, case["interleaved"], case["norm"])
                 for i, name in enumerate("qk"))


def _plain_attention(state):
    case = state["case"]
    hq, hk, D = case["hq"], case["hk"], case["D"]
    out = torch.empty_like(state["q"])
    q0 = k0 = 0
    for nq, nk in zip(state["q_lens"], state["kv_lens"]):
        # The rows of a group's heads stand one below the other against their shared keys: [hk, group * nq, nk].
        q = state["q"][q0:q0 + nq].float().view(nq, hk, hq // hk, D).permute(1, 2, 0, 3).reshape(hk, -1, D)
        k = state["k"][k0:k0 + nk].float().permute(1, 2, 0).contiguous()
        v = state["v"][k0:k0 + nk].float().permute(1, 0, 2).contiguous()
        s = torch.bmm(q, k).mul_(1.0 / math.sqrt(D))
        if case["causal"]:
            late = torch.arange(nk, device="cuda") > torch.arange(nq, device="cuda")[:, None] + (nk - nq)
            s.view(hk, hq // hk, nq, nk).masked_fill_(late, -torch.inf)
        s.sub_(s.amax(-1, keepdim=True)).exp_()
        o = torch.bmm(s, v) / s.sum(-1, keepdim=True)
        out[q0:q0 + nq] = o.view(hk, hq // hk, nq, D).permute(2, 0, 1, 3).reshape(nq, hq, D).to(out.dtype)
        q0, k0 = q0 + nq, k0 + nk
    return out


def _plain_adapters(state):
    out = state["y"].clone()
    for a, rows in state["rows"]:
        u = state["x"][rows].float() @ state["down"][a].float().t()
        delta = (u @ state["up"][a].float().t()).mul_(state["scale"][a])
        out[rows] = (state["y"][rows].float() + delta).to(out.dtype)
    return out


def run(state):
    op = state["case"]["op"]
    if not own:
        plain = {"qk_norm_rope": _plain_qk_norm_rope, "attention": _plain_attention, "adapters": _plain_adapters}
        return plain[op](state)
    import hyperflow_h3_flash_amd as hf

    if op == "qk_norm_rope":
        w = state["weights"]
        return hf.qk_norm_rope(state["q"], state["k"], state["positions"], state["rotary"],
                               q_weight=None if w is None else w[0], k_weight=None if w is None else w[1],
                               norm=w is not None, eps=1e-6)
    if op == "attention":
        return hf.packed_attention(state["q"], state["k"], state["v"], state["plan"])
    return hf.adapter_add(state["y"], state["x"], state["down"], state["up"], state["plan"], scale=state["scale"])


# -------------------------------------------------------------------------------------------------------- in 64 bits

def _exact_rope(case, state):
    """Each pair as a complex number, turned by exp(i position rate)."""
    rate, axis = [], []
    for a, dim in enumerate(_ints(case["axes"])):
        rate += [case["theta"] ** (-2.0 * i / dim) for i in range(dim // 2)]
        axis += [a] * (dim // 2)
    rate = torch.tensor(rate, device="cuda", dtype=torch.float64)
    phase = state["positions"][:, axis].double() * rate
    turn = torch.polar(torch.ones_like(phase), phase)[:, None, :]
    P = rate.numel()
    outputs = []
    for i, name in enumerate("qk"):
        x = state[name].double()
        if case["norm"]:
            x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * state["weights"][i].double()
        if case["interleaved"]:
            z = torch.view_as_complex(x[..., :2 * P].unflatten(-1, (P, 2)).contiguous()) * turn
            head = torch.view_as_real(z).flatten(-2)
        else:
            z = torch.complex(x[..., :P].contiguous(), x[..., P:2 * P].contiguous()) * turn
            head = torch.cat([z.real, z.imag], dim=-1)
        outputs.append(torch.cat([head, x[..., 2 * P:]], dim=-1))
    return tuple(outputs)


def _exact_attention(case, state):
    """One head of one sequence at a time, a few thousand rows of the scores at once."""
    out = torch.zeros(state["q"].shape, device="cuda", dtype=torch.float64)
    group = case["hq"] // case["hk"]
    q0 = k0 = 0
    for nq, nk in zip(state["q_lens"], state["kv_lens"]):
        for h in range(case["hq"]):
            k = state["k"][k0:k0 + nk, h // group].double().t().contiguous()
            v = state["v"][k0:k0 + nk, h // group].double().contiguous()
            for i in range(0, nq, 16384):
                n = min(16384, nq - i)
                s = (state["q"][q0 + i:q0 + i + n, h].double() @ k) / math.sqrt(case["D"])
                if case["causal"]:
                    s = s.masked_fill(torch.ones_like(s, dtype=torch.bool).triu(i + nk - nq + 1), -math.inf)
                out[q0 + i:q0 + i + n, h] = torch.softmax(s, dim=-1) @ v
        q0, k0 = q0 + nq, k0 + nk
    return out


def _exact_adapters(case, state):
    """One request at a time."""
    out = state["y"].double()
    m = 0
    for n, a in zip(state["lens"], state["ids"]):
        if a >= 0:
            u = state["x"][m:m + n].double() @ state["down"][a].double().t().contiguous()
            out[m:m + n] += state["scale"][a].double() * (u @ state["up"][a].double().t().contiguous())
        m += n
    return out


def exact(case, seed):
    state = _inputs(case, seed)
    forms = {"qk_norm_rope": _exact_rope, "attention": _exact_attention, "adapters": _exact_adapters}
    return forms[case["op"]](case, state)

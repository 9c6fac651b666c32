"""The performance cases of a transformer block's operators around its attention and of the 4-bit cache that its attention
reads: the norms before and after a block with its gate and residual, keys and values written to pages of 4-bit codes and
read back, attention over such pages, and copies of pages.

A case names one call (``op``) and its sizes; texts of comma-separated numbers are lengths, one a request:

* ``residual_norm``: rows [T, C] of packed requests: ``r = residual x + gate post(y)``, ``n = norm(r) w (1 + scale) + shift``.
* ``cache_write``: ``new`` tokens of each request behind the ``held`` ones of its cache, then the requests' whole keys and
  values out of the pages, as packed attention takes them.
* ``cached_attention``: queries of packed requests against their caches.
* ``copy_pages``: pages of all layers copied within the pool, as a fork or a compaction does.

A page holds ``page`` tokens of one layer. Codes are the 4-bit floats 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives, times a
power of two for each 32 channels of a head: the least one, within the limits of ``SCALES``, that is at least a seventh of
the largest magnitude. Ties go to the even code, values past 6 to 6.

``run`` computes them in plain fp32 torch operations, or with ``own`` set through this framework's entry points.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
#: The least and largest exponent of a group's scale, by the type of the keys and values.
SCALES = {"bf16": (-125, 125), "fp16": (-23, 13)}
GROUP = 32
EPS = 1e-6
#: Limits of a drawn case, by the listed ones: bytes of a norm, multiply-adds x 2 of an attention, tokens x channels of
#: written caches, bytes of a pool.
MOST_BYTES = 1.63e9
MOST_FLOPS = 4.0 * 4860 * 37710 * 7 * 128
MOST_CACHED = 2.0e8
MOST_POOL = 1.3e9


def _ints(text):
    return [int(v) for v in text.split(",")]


def _text(values):
    return ",".join(str(v) for v in values)


def _norm_case(name, lens, C, norm, post, y=True, weights=False, modulated=True, residual=1.0, stream="bf16",
               dtype="bf16"):
    return {"name": name, "op": "residual_norm", "lens": lens, "C": C, "norm": norm, "post": post, "y": y,
            "weights": weights, "modulated": modulated, "residual": residual, "stream": stream, "dtype": dtype}


def _write_case(name, new, held, hk, D, page=64, dtype="bf16"):
    return {"name": name, "op": "cache_write", "new": new, "held": held, "hk": hk, "D": D, "page": page, "dtype": dtype}


def _cached_case(name, q_lens, kv_lens, hq, hk, D, causal, page=64, dtype="bf16"):
    return {"name": name, "op": "cached_attention", "q_lens": q_lens, "kv_lens": kv_lens, "hq": hq, "hk": hk, "D": D,
            "causal": causal, "page": page, "dtype": dtype}


def _copy_case(name, layers, pages, moves, page_bytes):
    return {"name": name, "op": "copy_pages", "layers": layers, "pages": pages, "moves": moves, "page_bytes": page_bytes}


def listed():
    return [
        # Between attention and feed-forward of the model's 5.2 s clip: gated residual and the next modulated norm.
        _norm_case("norm_clip", "37710", 5376, "layer", "none"),
        # Clips and images of several requests packed in one batch, each with its own modulation; norms with weights
        # before and after the branch, the residual stream in float32.
        _norm_case("norm_packed", "5168,1001,2600,77", 5120, "rms", "rms", weights=True, stream="fp32"),
        # One new token of each of a few requests: launch latency.
        _norm_case("norm_rows", "1,1,1,1,1,1,1", 5120, "rms", "none", weights=True, modulated=False, residual=0.5,
                   dtype="fp16", stream="fp16"),
        # Prompts of a text encoder filling their caches.
        _write_case("write_prompts", "4099,1537,300,61,2048", "0,0,0,0,0", 8, 128),
        # One new token of each of sixteen requests behind short caches.
        _write_case("write_tokens", _text([1] * 16), _text([63, 64, 733, 0, 512, 250, 61, 127, 99, 300, 31, 77, 640, 201,
                                                            125, 50]), 8, 128),
        # Serving: one new token of each request against its own cache.
        _cached_case("cached_tokens", _text([1] * 16), _text([8191, 4096, 733, 1, 16384, 2500, 6001, 127, 9999, 3000, 512,
                                                              7777, 64, 12001, 1025, 5000]), 32, 8, 128, True),
        # One request with a very long cache.
        _cached_case("cached_long", "1", "131072", 64, 8, 128, True, page=128),
        # One new token of a small decoder: the smallest call.
        _cached_case("cached_short", "1", "77", 12, 12, 64, True, page=32, dtype="fp16"),
        # Prompts' last parts against all that is cached of them, and one new token among them.
        _cached_case("cached_prompts", "512,300,61,1", "4096,8191,733,2500", 32, 8, 128, True),
        # A clip extended by three latent frames, one GPU's heads under an 8-way head split: the largest.
        _cached_case("cached_clip", "4860", "37710", 7, 7, 128, False),
        # A request forked: its last, partly filled page copied in every layer, for eight continuations.
        _copy_case("pages_fork", 47, 64, 8, 64 * 8 * 136),
        # A pool compacted: a third of its pages moved to the front, all layers.
        _copy_case("pages_compact", 47, 384, 128, 64 * 8 * 136),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["residual_norm", "cache_write", "cached_attention", "cached_attention", "cached_attention",
                     "copy_pages"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    while True:
        if op == "residual_norm":
            count = _log_int(rng, 1, 16)
            longest = _log_int(rng, 1, 38000 // count)
            lens = [_log_int(rng, max(1, longest // 8), longest) for _ in range(count)]
            y = rng.random() < 0.8
            case = _norm_case("", _text(lens), 8 * _log_int(rng, 32, 1024), rng.choice(["rms", "layer"]),
                              rng.choice(["none", "none", "rms", "layer"]) if y else "none", y, rng.random() < 0.5,
                              rng.random() < 0.6, rng.choice([1.0, 1.0, 0.5]) if y else 1.0,
                              rng.choice([dtype, dtype, "fp32"]), dtype)
            fits = work(case)["bytes"] <= MOST_BYTES
        elif op == "copy_pages":
            pages = _log_int(rng, 8, 2000)
            case = _copy_case("", rng.randint(1, 60), pages, _log_int(rng, 1, pages // 2),
                              rng.choice([32, 64, 128]) * rng.choice([1, 2, 4, 7, 8, 12]) * rng.choice([36, 72, 104, 136]))
            fits = case["layers"] * pages * case["page_bytes"] <= MOST_POOL
        else:
            D = rng.choice([64, 80, 96, 128, 128, 128])
            hk = rng.choice([1, 2, 4, 7, 8, 12])
            page = rng.choice([32, 64, 64, 128])
            count = _log_int(rng, 1, 24)
            longest = _log_int(rng, 16, 24000)
            held = [max(1, min(longest, _log_int(rng, max(1, longest // 16), longest))) for _ in range(count)]
            if op == "cache_write":
                new = [1] * count if rng.random() < 0.5 else [_log_int(rng, 1, 4000) for _ in range(count)]
                case = _write_case("", _text(new), _text([v - 1 for v in held]), hk, D, page, dtype)
                fits = (sum(held) + sum(new)) * hk * D <= MOST_CACHED
            else:
                hq = hk * rng.choice([1, 1, 2, 4, 5, 8])
                form = rng.choice(["tokens", "tokens", "few", "tail", "cross"])
                if form == "tokens":
                    q = [1] * count
                elif form == "few":  # a few tokens proposed and judged at once
                    q = [min(v, rng.randint(1, 8)) for v in held]
                elif form == "tail":
                    q = [_log_int(rng, 1, v) for v in held]
                else:
                    q = [_log_int(rng, 16, 4000) for _ in range(count)]
                case = _cached_case("", _text(q), _text(held), hq, hk, D, form != "cross" and rng.random() < 0.7, page,
                                    dtype)
                fits = (sum(4.0 * D * hq * a * b for a, b in zip(q, held)) <= MOST_FLOPS
                        and sum(held) * hk * D <= MOST_CACHED and sum(q) * hq * D <= MOST_CACHED)
        if fits:
            del case["name"]
            return case


def _cached_bytes(tokens, hk, D):
    """Codes and scales of keys and values."""
    return 2 * tokens * hk * (D // 2 + -(-D // GROUP))


def work(case):
    if case["op"] == "residual_norm":
        T, C = sum(_ints(case["lens"])), case["C"]
        wide = 4 if case["stream"] == "fp32" else 2
        passes = wide + 2 + ((wide + 2) if case["y"] else 0)
        vectors = (3 if case["y"] else 2) * len(_ints(case["lens"])) if case["modulated"] else 0
        vectors += (case["post"] != "none") + 1 if case["weights"] else 0
        return {"bytes": T * C * passes + 2 * vectors * C, "flops": 12 * T * C}
    if case["op"] == "cache_write":
        new, held, hk, D = sum(_ints(case["new"])), sum(_ints(case["held"])), case["hk"], case["D"]
        return {"bytes": 4 * new * hk * D + _cached_bytes(new, hk, D) + _cached_bytes(new + held, hk, D)
                + 4 * (new + held) * hk * D, "flops": 8 * new * hk * D + 2 * (new + held) * hk * D}
    if case["op"] == "cached_attention":
        q, kv, D = _ints(case["q_lens"]), _ints(case["kv_lens"]), case["D"]
        if case["causal"]:  # row i of a sequence sees i + 1 + (kv - q) keys
            pairs = sum(sum(min(max(i + 1 + b - a, 0), b) for i in range(a)) for a, b in zip(q, kv))
        else:
            pairs = sum(a * b for a, b in zip(q, kv))
        return {"bytes": 4 * D * sum(q) * case["hq"] + _cached_bytes(sum(kv), case["hk"], D),
                "flops": 4 * D * case["hq"] * pairs}
    return {"bytes": 2 * case["layers"] * case["moves"] * case["page_bytes"], "flops": 0}


# ------------------------------------------------------------------------------------------------------------- inputs

def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _inputs(case, seed):
    """The inputs of a case, from the seed alone, as tensors and plain values."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "residual_norm":
        lens, C = _ints(case["lens"]), case["C"]
        T, dtype = sum(lens), DTYPES[case["dtype"]]
        # A residual stream as deep blocks see it: a mean, and a few channels far stronger than the others.
        x = 2 * _normal(gen, T, C) + 0.3 * _normal(gen, C)
        x[:, ::199] *= 10
        inputs = {"lens": lens, "x": x.to(DTYPES[case["stream"]]),
                  "y": (_normal(gen, T, C) + 0.1).to(dtype) if case["y"] else None,
                  "w": None, "pw": None, "modulation": None}
        if case["weights"]:
            inputs["w"] = (1 + 0.2 * _normal(gen, C)).to(dtype)
            inputs["pw"] = (1 + 0.2 * _normal(gen, C)).to(dtype) if case["post"] != "none" else None
        if case["modulated"]:  # gate, scale and shift as slices of one projection's output
            inputs["modulation"] = (0.4 * _normal(gen, len(lens), 3, C)).to(dtype)
        return inputs
    if case["op"] == "copy_pages":
        pool = torch.randint(0, 256, (case["layers"], case["pages"], case["page_bytes"]), generator=gen, device="cuda",
                             dtype=torch.uint8)
        order = torch.randperm(case["pages"], generator=torch.Generator().manual_seed(seed)).tolist()
        n = case["moves"]
        return {"pool": pool, "src": order[:n], "dst": order[n:2 * n]}
    dtype, hk, D = DTYPES[case["dtype"]], case["hk"], case["D"]
    write = case["op"] == "cache_write"
    if write:
        held, new = _ints(case["held"]), _ints(case["new"])
        total = [a + b for a, b in zip(held, new)]
    else:
        total = _ints(case["kv_lens"])
    # Keys with a few strong channels, as rotated keys have; values with a mean of their own per channel. Both are views of
    # a fused projection's output.
    hq = case.get("hq", hk)
    k = 1.2 * _normal(gen, sum(total), hk, D) * (1 + (torch.arange(D, device="cuda") % 29 == 3))
    v = _normal(gen, sum(total), hk, D) + 0.5 * _normal(gen, hk, D)
    wide = torch.zeros(sum(total), 2 * hk, D, device="cuda", dtype=dtype)
    wide[:, :hk], wide[:, hk:] = k, v
    inputs = {"k": wide[:, :hk], "v": wide[:, hk:], "total": total}
    if write:
        inputs["held"] = held
        fresh = torch.cat([torch.arange(a + b) >= a for a, b in zip(held, new)]).cuda()
        inputs["wide"], inputs["fresh"] = wide, fresh
    else:
        inputs["q"] = _normal(gen, sum(_ints(case["q_lens"])), hq, D).to(dtype)
    return inputs


def prepare(case, seed):
    state = {"case": case, **_inputs(case, seed)}
    op = case["op"]
    if op == "residual_norm":
        lens, C = state["lens"], case["C"]
        m = state.pop("modulation")
        for i, name in enumerate(("gate", "shift", "scale")):
            state[name] = None if m is None else m[:, i]
        if not case["y"]:
            state["gate"] = None
        if own:
            import hyperflow_h3_flash_amd as hf

            state["rows"] = hf.RowPlan(lens, device="cuda") if case["modulated"] else None
        else:
            state["rows"] = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens)).cuda()
        return state
    if op == "copy_pages":
        if not own:
            state["src"], state["dst"] = (torch.tensor(state[name], device="cuda") for name in ("src", "dst"))
        return state
    held = state["held"] if op == "cache_write" else state["total"]
    if op == "cache_write":  # what is held is in the cache, what is new lies packed behind one another
        fresh, wide, hk = state.pop("fresh"), state.pop("wide"), case["hk"]
        old, new = wide[~fresh], wide[fresh]
        state["k"], state["v"] = new[:, :hk], new[:, hk:]
        k, v = old[:, :hk], old[:, hk:]
    else:
        k, v = state.pop("k"), state.pop("v")
    pages = sum(-(-n // case["page"]) for n in state["total"])
    if own:
        import hyperflow_h3_flash_amd as hf

        cache = hf.KVCache(1, case["hk"], case["D"], pages, page_size=case["page"], dtype=DTYPES[case["dtype"]],
                           device="cuda")
        requests = [cache.new() for _ in held]
        # Each request's first half, then its second: pages of one request do not lie side by side, as in a server's pool.
        first = torch.cat([torch.arange(n) < n // 2 for n in held]).cuda()
        for half, lens in ((first, [n // 2 for n in held]), (~first, [n - n // 2 for n in held])):
            hf.cache_append(cache, 0, k[half], v[half], cache.plan(requests, lens, heads=case["hk"]))
        state["cache"] = cache
        if op == "cache_write":
            state["plan"] = cache.plan(requests, _ints(case["new"]), heads=case["hk"])
        else:
            state["plan"] = cache.plan(requests, _ints(case["q_lens"]), new_lengths=[0] * len(held), heads=case["hq"],
                                       causal=case["causal"])
        return state
    # The plain form's cache: the same pages, in a random order; a token's codes and scales side by side.
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))
    slots = (order[:, None] * case["page"] + torch.arange(case["page"])).flatten()
    table, at = [], 0
    for n in state["total"]:
        table.append(slots[at * case["page"]:at * case["page"] + n])
        at += -(-n // case["page"])
    G = -(-case["D"] // GROUP)
    state["codes"] = torch.zeros(pages * case["page"], 2, case["hk"], G, GROUP // 2, device="cuda", dtype=torch.uint8)
    state["scales"] = torch.zeros(pages * case["page"], 2, case["hk"], G, device="cuda", dtype=torch.uint8)
    state["table"] = torch.cat(table).cuda()
    state["into"] = torch.cat([t[n:] for t, n in zip(table, held)]).cuda()
    _plain_write(state, torch.cat([t[:n] for t, n in zip(table, held)]).cuda(), k, v)
    return state


# --------------------------------------------------------------------------------------------------- the plain forms

def _plain_norm(h, kind, weight):
    if kind == "layer":
        h = h - h.mean(-1, keepdim=True)
    if kind != "none":
        h = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS)
    return h if weight is None else h * weight.float()


def _plain_residual_norm(state):
    case, rows = state["case"], state["rows"]
    r = state["x"].float()
    outputs = []
    if case["y"]:
        branch = _plain_norm(state["y"].float(), case["post"], state["pw"])
        if case["modulated"]:
            branch = branch * state["gate"].float()[rows]
        r = case["residual"] * r + branch
        outputs.append(r.to(state["x"].dtype))
    n = _plain_norm(r, case["norm"], state["w"])
    if case["modulated"]:
        n = n * (1 + state["scale"].float()[rows]) + state["shift"].float()[rows]
    return (*outputs, n.to(DTYPES[case["dtype"]]))


def _plain_quantize(x, dtype):
    """(packed codes [..., G, 16], scale bytes [..., G]) of x [..., D]."""
    G = -(-x.shape[-1] // GROUP)
    h = torch.nn.functional.pad(x.float(), (0, G * GROUP - x.shape[-1])).unflatten(-1, (G, GROUP))
    m, e = torch.frexp(h.abs().amax(-1))
    e = (e - torch.where(m <= 0.875, 3, 2)).clamp(*SCALES[dtype])
    a = torch.ldexp(h.abs(), -e[..., None])
    code = torch.zeros_like(a, dtype=torch.uint8)
    for border, even in ((0.25, True), (0.75, False), (1.25, True), (1.75, False), (2.5, True), (3.5, False), (5.0, True)):
        code += (a > border) if even else (a >= border)
    code |= torch.signbit(h).to(torch.uint8) << 3
    return code[..., 0::2] | (code[..., 1::2] << 4), (e + 127).to(torch.uint8)


def _plain_write(state, slots, k, v):
    for i, t in enumerate((k, v)):
        codes, scales = _plain_quantize(t, state["case"]["dtype"])
        state["codes"][slots, i] = codes
        state["scales"][slots, i] = scales


def _plain_read(state, slots, which):
    """[tokens, heads, D] in fp32."""
    codes, D = state["codes"][slots, which], state["case"]["D"]
    levels = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device="cuda")
    levels = torch.cat([levels, -levels])
    h = levels[torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2).long()]
    h = torch.ldexp(h, state["scales"][slots, which][..., None].int() - 127)
    return h.flatten(-2)[..., :D]


def _plain_cache_write(state):
    _plain_write(state, state["into"], state["k"], state["v"])
    dtype = DTYPES[state["case"]["dtype"]]
    return tuple(_plain_read(state, state["table"], i).to(dtype) for i in range(2))


def _plain_cached_attention(state):
    case = state["case"]
    hq, hk, D = case["hq"], case["hk"], case["D"]
    out = torch.empty_like(state["q"])
    q0 = k0 = 0
    for nq, nk in zip(_ints(case["q_lens"]), state["total"]):
        slots = state["table"][k0:k0 + nk]
        # The rows of a group's heads stand one below the other against their shared keys: [hk, group * nq, nk].
        q = state["q"][q0:q0 + nq].float().view(nq, hk, hq // hk, D).permute(1, 2, 0, 3).reshape(hk, -1, D)
        k = _plain_read(state, slots, 0).permute(1, 2, 0).contiguous()
        v = _plain_read(state, slots, 1).permute(1, 0, 2).contiguous()
        s = torch.bmm(q, k).mul_(1.0 / math.sqrt(D))
        if case["causal"]:
            late = torch.arange(nk, device="cuda") > torch.arange(nq, device="cuda")[:, None] + (nk - nq)
            s.view(hk, hq // hk, nq, nk).masked_fill_(late, -torch.inf)
        s.sub_(s.amax(-1, keepdim=True)).exp_()
        o = torch.bmm(s, v) / s.sum(-1, keepdim=True)
        out[q0:q0 + nq] = o.view(hk, hq // hk, nq, D).permute(2, 0, 1, 3).reshape(nq, hq, D).to(out.dtype)
        q0, k0 = q0 + nq, k0 + nk
    return out


def _plain_copy_pages(state):
    state["pool"][:, state["dst"]] = state["pool"][:, state["src"]]
    return state["pool"]


def run(state):
    case = state["case"]
    op = case["op"]
    if not own:
        plain = {"residual_norm": _plain_residual_norm, "cache_write": _plain_cache_write,
                 "cached_attention": _plain_cached_attention, "copy_pages": _plain_copy_pages}
        return plain[op](state)
    import hyperflow_h3_flash_amd as hf

    if op == "residual_norm":
        r, n = hf.residual_norm(state["x"], state["y"], rows=state["rows"], residual=case["residual"],
                                gate=state["gate"], post_norm=None if case["post"] == "none" else case["post"],
                                post_weight=state["pw"], norm=case["norm"], weight=state["w"], scale=state["scale"],
                                shift=state["shift"], eps=EPS, dtype=DTYPES[case["dtype"]])
        return (r, n) if case["y"] else (n,)
    if op == "cache_write":
        hf.cache_append(state["cache"], 0, state["k"], state["v"], state["plan"])
        return hf.cache_read(state["cache"], 0, state["plan"])
    if op == "cached_attention":
        return hf.cached_attention(state["q"], state["cache"], 0, state["plan"])
    return hf.copy_pages(state["pool"], state["src"], state["dst"])


# -------------------------------------------------------------------------------------------------------- in 64 bits

def _exact_normed(h, kind, weight):
    if kind == "none":
        return h
    mean = h.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(h[..., :1])
    spread = torch.sqrt(((h - mean) ** 2).mean(-1, keepdim=True) + EPS)
    return (h - mean) / spread * (1.0 if weight is None else weight.double())


def _exact_residual_norm(case, state):
    """One request at a time, a few thousand rows at once."""
    r = state["x"].double() if case["y"] else None
    n = torch.empty(state["x"].shape, device="cuda", dtype=torch.float64)
    at = 0
    for i, length in enumerate(state["lens"]):
        gate, shift, scale = state["modulation"][i].double() if case["modulated"] else (1.0, 0.0, 0.0)
        for a in range(at, at + length, 4096):
            b = min(a + 4096, at + length)
            h = state["x"][a:b].double()
            if case["y"]:
                h = case["residual"] * h + gate * _exact_normed(state["y"][a:b].double(), case["post"], state["pw"])
                r[a:b] = h
            n[a:b] = _exact_normed(h, case["norm"], state["w"]) * (1 + scale) + shift
        at += length
    return (r, n) if case["y"] else (n,)


def _exact_codes(x, dtype):
    """The values that x [tokens, heads, D] is held as: each magnitude's nearest multiple among the levels."""
    tokens, heads, D = x.shape
    low, high = SCALES[dtype]
    levels = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device="cuda", dtype=torch.float64)
    middle = (levels[1:] + levels[:-1]) / 2
    out = torch.empty(x.shape, device="cuda", dtype=torch.float64)
    for c in range(0, D, GROUP):
        h = x[..., c:c + GROUP].double()
        top = h.abs().amax(-1, keepdim=True)
        s = 2.0 ** torch.ceil(torch.log2(top / 7)).clamp(low, high)
        a = (h.abs() / s).contiguous()
        below = torch.searchsorted(middle, a)  # the lower level where a is a middle, else the nearest
        above = torch.searchsorted(middle, a, right=True)
        nearest = levels[torch.where(below % 2 == 0, below, above)]
        out[..., c:c + GROUP] = torch.sign(h) * nearest * s
    return out


def _exact_cached_attention(case, state):
    """One head of one sequence at a time."""
    k_all, v_all = _exact_codes(state["k"], case["dtype"]), _exact_codes(state["v"], case["dtype"])
    out = torch.zeros(state["q"].shape, device="cuda", dtype=torch.float64)
    group = case["hq"] // case["hk"]
    q0 = k0 = 0
    for nq, nk in zip(_ints(case["q_lens"]), state["total"]):
        for h in range(case["hq"]):
            k = k_all[k0:k0 + nk, h // group].t().contiguous()
            v = v_all[k0:k0 + nk, h // group].contiguous()
            for i in range(0, nq, 8192):
                n = min(8192, nq - i)
                s = (state["q"][q0 + i:q0 + i + n, h].double() @ k) / math.sqrt(case["D"])
                if case["causal"]:
                    s = s.masked_fill(torch.ones_like(s, dtype=torch.bool).triu(i + nk - nq + 1), -math.inf)
                out[q0 + i:q0 + i + n, h] = torch.softmax(s, dim=-1) @ v
        q0, k0 = q0 + nq, k0 + nk
    return out


def exact(case, seed):
    state = _inputs(case, seed)
    if case["op"] == "residual_norm":
        return _exact_residual_norm(case, state)
    if case["op"] == "cache_write":
        return tuple(_exact_codes(state[name], case["dtype"]) for name in "kv")
    if case["op"] == "cached_attention":
        return _exact_cached_attention(case, state)
    for s, d in zip(state["src"], state["dst"]):  # a page of all layers at a time
        state["pool"][:, d] = state["pool"][:, s].clone()
    return state["pool"]

"""The 4-bit cache on the host: its values, its accounts, its plans and what it refuses."""

from __future__ import annotations

import copy
import ctypes
import os
import pickle
import random
import re
import struct

import numpy as np
import pytest
import torch

import block_utils as U
import cache_utils as C
from hyperflow_h3_flash_amd import (KVCache, RowPlan, _native, cache_append, cache_read, cached_attention, copy_pages,
                                    residual_norm)

BF, HF = torch.bfloat16, torch.float16
HEADER = os.path.join(_native.REPO_DIR, "include", "hf_cache.h")


def rnd(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_native.BLOCK_LIB_PATH):
        pytest.fail(f"{_native.BLOCK_LIB_PATH} not built: run __graft_entry__.build()")
    return _native.block_library()


# --------------------------------------------------------------------------------------------------------------- values

@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [16, 48, 96, 128])
def test_values_are_the_nearest_levels(D, dtype):
    k = torch.ldexp(rnd(1, 70, 2, D), torch.randint(-8, 9, (70, 2, 1), generator=torch.Generator().manual_seed(2))).to(dtype)
    v = (torch.randint(-28, 29, (70, 2, D), generator=torch.Generator().manual_seed(3)) / 4).to(dtype)  # ties among them
    cache = KVCache(2, 2, D, 3, page_size=32, dtype=dtype, device="cpu")
    plan = cache.plan([cache.new()], [70])
    cache_append(cache, 1, k, v, plan)
    got = cache_read(cache, 1, plan)
    assert torch.equal(got[0].double(), C.held(k)) and torch.equal(got[1].double(), C.held(v))
    assert cache.data[0].eq(0).all()


def test_ties_limits_and_groups_that_are_not_finite():
    x = torch.zeros(1, 1, 32)
    x[0, 0, :10] = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -5.0])
    y = torch.zeros(1, 1, 32)
    y[0, 0, :3] = torch.tensor([7.0, 7.0 * 2 ** -10, -3.0])  # 7 stays at a scale of 1, and is read as 6
    cache = KVCache(1, 1, 32, 1, dtype=BF, device="cpu")
    plan = cache.plan([cache.new()], [1])
    cache_append(cache, 0, x.to(BF), y.to(BF), plan)
    k, v = cache_read(cache, 0, plan)
    assert k[0, 0, :10].tolist() == [6.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 0.0, -4.0]
    assert v[0, 0, :3].tolist() == [6.0, 0.0, -3.0]
    for dtype in (BF, HF):
        top = torch.finfo(dtype).max
        z = torch.tensor([top, torch.inf]).to(dtype).view(2, 1, 1).repeat(1, 1, 32)
        cache = KVCache(1, 1, 32, 1, dtype=dtype, device="cpu")
        plan = cache.plan([cache.new()], [2])
        cache_append(cache, 0, z, z, plan)
        k, _ = cache_read(cache, 0, plan)
        assert k[0].eq(6.0 * 2.0 ** C.LIMITS[dtype][1]).all() and k[1].isnan().all()


def scale_bytes(cache, page, head, token):
    """The scale bytes of a token's keys and values as the header lays them out, on the host."""
    G, P = -(-cache.head_dim // 32), cache.page_size
    S = 4 if G == 3 else G
    slab = cache.data[0, page].view(cache.kv_heads, -1)[head]
    at = 2 * G * P * 16 + token * 2 * S
    return slab[at:at + G].tolist(), slab[at + S:at + S + G].tolist()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("dtype,least,most", [(BF, 2, 252), (HF, 104, 140)])
@pytest.mark.parametrize("D", [16, 80, 128])
def test_scales_are_the_headers(D, dtype, least, most, device):
    """The least power of two that is a seventh of the largest, within the type's limits, and 2^-3 (byte 124) for zeros."""
    text = " ".join(open(HEADER).read().replace("*", " ").split())
    assert "2^-3 for a group of zeros" in text and "e from -125 to 125 for bfloat16 and -23 to 13 for float16" in text
    tiny, top = torch.finfo(dtype).smallest_normal * 2.0 ** -7, torch.finfo(dtype).max
    k = torch.zeros(5, 1, D)
    v = torch.zeros(5, 1, D)
    v[1, 0, 3], v[2, 0, 3], v[3, 0, 3], v[4, 0, 3] = tiny, top, 7.0, 7.0 * (1 + 2.0 ** -6)
    k[4, 0] = -0.0
    k, v = k.to(dtype).to(device), v.to(dtype).to(device)
    cache = KVCache(1, 1, D, 1, page_size=32, dtype=dtype, device=device)
    cache_append(cache, 0, k, v, cache.plan([cache.new()], [5]))
    G = -(-D // 32)
    for token, first in enumerate((124, least, most, 127, 128)):
        assert scale_bytes(cache, 0, 0, token) == ([124] * G, [first] + [124] * (G - 1))


@pytest.mark.parametrize("causal", [False, True])
def test_host_attention(causal):
    q_lens, kv_lens = [1, 9, 0, 40], [70, 9, 33, 31]
    cache = KVCache(1, 2, 48, 8, page_size=32, dtype=BF, device="cpu")
    requests = [cache.new() for _ in kv_lens]
    k, v, q = rnd(1, sum(kv_lens), 2, 48).to(BF), rnd(2, sum(kv_lens), 2, 48).to(BF), rnd(3, sum(q_lens), 6, 48).to(BF)
    cache_append(cache, 0, k, v, cache.plan(requests, kv_lens))
    plan = cache.plan(requests, q_lens, new_lengths=[0] * 4, heads=6, causal=causal)
    ref, bound = C.attention(q, k, v, q_lens, kv_lens, causal, 48 ** -0.5)
    out = torch.empty_like(q)
    assert cached_attention(q, cache, 0, plan, out=out) is out
    U.check(out, ref, bound)


# ------------------------------------------------------------------------------------------------------------- accounts

@pytest.mark.parametrize("seed", range(4))
def test_any_order_of_steps_forks_and_moves_keeps_every_token(seed):
    """Against a model that keeps each request's tokens in a list."""
    rng = random.Random(seed)
    cache = KVCache(2, 1, 16, 24, page_size=32, device="cpu")
    model: dict[int, list[int]] = {}
    counter = 0

    def token(i):  # values that are held exactly, by token
        return torch.tensor([float(1 + i % 3)] + [float(i >> b & 1) for b in range(15)]).to(BF).view(1, 1, 16)

    for _ in range(150):
        what = rng.choice(["new", "step", "step", "step", "step", "fork", "truncate", "free", "compact"])
        if what == "new" or not model:
            if len(model) < 6:
                model[cache.new()] = []
            continue
        request = rng.choice(list(model))
        if what == "step":
            some = rng.sample(list(model), rng.randint(1, len(model)))
            new = [rng.choice([0, 1, 1, 5, 31, 40]) for _ in some]
            before = copy.deepcopy([(r, cache.table(r), cache.length(r)) for r in model]), cache.free_pages
            try:
                plan = cache.plan(some, [1] * len(some), new_lengths=new)
            except RuntimeError:
                assert before == ([(r, cache.table(r), cache.length(r)) for r in model], cache.free_pages)
                continue
            ids = []
            for r, n in zip(some, new):
                mine = list(range(counter, counter + n))
                counter += n
                model[r] += mine
                ids += mine
            rows = torch.cat([token(i) for i in ids]) if ids else torch.empty(0, 1, 16, dtype=BF)
            for layer in range(2):
                cache_append(cache, layer, rows, -rows, plan)
        elif what == "fork" and len(model) < 6:
            model[cache.fork(request)] = list(model[request])
        elif what == "truncate":
            n = rng.randint(0, len(model[request]))
            cache.truncate(request, n)
            del model[request][n:]
        elif what == "free":
            cache.free(request)
            del model[request]
        elif what == "compact":
            used = cache.compact()
            assert used == cache.pages - cache.free_pages
            assert all(p < used for r in model for p in cache.table(r))
        pages = {p for r in model for p in cache.table(r)}
        assert cache.free_pages == cache.pages - len(pages)
        assert cache._uses == [sum(cache.table(r).count(p) for r in model) for p in range(cache.pages)]
        live = list(model)
        plan = cache.plan(live, [0] * len(live))
        want = [token(i) for r in live for i in model[r]]
        for layer in range(2):
            k, v = cache_read(cache, layer, plan)
            assert torch.equal(k, torch.cat(want) if want else k[:0]) and torch.equal(v, -k)


def test_old_plans_are_refused_where_they_would_be_wrong():
    cache = KVCache(1, 1, 16, 8, page_size=32, device="cpu")
    a, b = cache.new(), cache.new()
    k = rnd(1, 40, 1, 16).to(BF)
    first = cache.plan([a], [40])
    cache_append(cache, 0, k, k, first)
    other = cache.plan([b], [40])
    second = cache.plan([a], [1])
    for plan in (first, other):  # longer requests do no harm
        cache_append(cache, 0, k, k, plan)
        cache_read(cache, 0, plan)
    c = cache.fork(a)
    with pytest.raises(ValueError, match="forked"):
        cache_append(cache, 0, k, k, first)
    with pytest.raises(ValueError, match="forked"):
        cache_append(cache, 0, k[:1], k[:1], second)
    cache_append(cache, 0, k, k, other)
    cache_read(cache, 0, first)
    cache.plan([c], [1])  # c's last page is its own now; a's plans are as good as before
    cache_read(cache, 0, second)
    cache.plan([a], [1])
    cache.truncate(a, 5)
    for plan in (first, second):
        with pytest.raises(ValueError, match="given back or moved"):
            cache_read(cache, 0, plan)
    last = cache.plan([b], [0])
    cache.free(a)
    cache_read(cache, 0, last)
    cache.free(b)
    with pytest.raises(ValueError, match="given back or moved"):
        cached_attention(torch.zeros(0, 1, 16, dtype=BF), cache, 0, last)
    with pytest.raises(ValueError, match="no request"):
        cache.length(a)
    with pytest.raises(ValueError, match="another cache"):
        cache_read(KVCache(1, 1, 16, 8, page_size=32, device="cpu"), 0, last)
    assert copy.copy(last) is last and copy.deepcopy(last) is last
    with pytest.raises(TypeError):
        pickle.dumps(last)


def test_a_step_that_does_not_fit_changes_nothing():
    cache = KVCache(1, 1, 16, 3, page_size=32, device="cpu")
    a = cache.new()
    cache.plan([a], [40])
    b = cache.fork(a)
    with pytest.raises(RuntimeError, match="2 pages, 1 of 3 are free"):
        cache.plan([a, b], [30, 1])
    assert cache.length(a) == cache.length(b) == 40 and cache.free_pages == 1
    cache.plan([a, b], [1, 1])  # one copy: the other keeps the page
    assert cache.free_pages == 0 and cache.table(a)[1] != cache.table(b)[1]


def test_a_step_costs_its_own_pages_not_the_pools():
    """A step that takes 16 pages compares page numbers on the way of 16 of a heap, not once for each free page."""
    compared = 0

    class Page(int):
        def __lt__(self, other):
            nonlocal compared
            compared += 1
            return int(self) < int(other)

    cache = KVCache(1, 1, 16, 1 << 16, page_size=32, device="cpu")
    requests = [cache.new() for _ in range(16)]
    cache._unused = [Page(p) for p in cache._unused]
    cache.plan(requests, [1] * 16)
    assert [cache.table(r) for r in requests] == [[i] for i in range(16)]
    assert compared <= 16 * 2 * 17  # two a level, 2^16 pages


def test_a_request_read_twice_beside_one_that_gets_tokens():
    cache = KVCache(1, 1, 16, 8, page_size=32, device="cpu")
    a = cache.new()
    k = rnd(1, 41, 1, 16).to(BF)
    cache_append(cache, 0, k[:40], k[:40], cache.plan([a], [40]))
    b = cache.fork(a)
    plan = cache.plan(iter([a, b, a]), [1, 1, 1], new_lengths=[0, 1, 0])
    cache_append(cache, 0, k[40:], k[40:], plan)
    got, _ = cache_read(cache, 0, plan)
    assert torch.equal(got.double(), C.held(torch.cat([k[:40], k, k[:40]])))
    for requests, new in (([a, b, a], [0, 0, 1]), ([a, a], [1, 1]), (iter([a, a]), [1, 0])):
        with pytest.raises(ValueError, match="named twice"):
            cache.plan(requests, [1] * len(new), new_lengths=new)
    assert cache.length(a) == 40 and cache.length(b) == 41 and cache.free_pages == 5


@pytest.mark.parametrize("broken", ["CachePlan", "copy_pages"])
def test_a_step_that_fails_while_it_is_built_changes_nothing(monkeypatch, broken):
    from hyperflow_h3_flash_amd import kv_cache

    def fail(*args, **kwargs):
        raise MemoryError("no")

    cache = KVCache(1, 1, 16, 9, page_size=32, device="cpu")
    a = cache.new()
    cache.plan([a], [40])
    b = cache.fork(a)
    tables = cache.table(a), cache.table(b)
    with monkeypatch.context() as m:
        m.setattr(kv_cache, broken, fail)
        with pytest.raises(MemoryError):
            cache.plan([a, b], [40, 1])
    assert (cache.table(a), cache.table(b)) == tables and cache.free_pages == 7 and cache.length(a) == cache.length(b) == 40
    cache.plan([a, b], [40, 1])
    assert cache.table(a) == [0, 2, 3] and cache.table(b) == [0, 1]


def test_refusals():
    for bad in (dict(layers=0), dict(kv_heads=0), dict(head_dim=24), dict(head_dim=144), dict(page_size=48), dict(pages=-1),
                dict(dtype=torch.float32), dict(pages=1 << 26)):
        args = dict(layers=1, kv_heads=1, head_dim=16, pages=2) | bad
        with pytest.raises(ValueError):
            KVCache(args.pop("layers"), args.pop("kv_heads"), args.pop("head_dim"), args.pop("pages"), device="cpu", **args)
    cache = KVCache(2, 2, 16, 4, device="cpu")
    a = cache.new()
    for bad in (lambda: cache.plan([a], [1, 2]), lambda: cache.plan([a], [-1]), lambda: cache.plan([a, a], [1, 1]),
                lambda: cache.plan([7], [1]), lambda: cache.plan([a], [1], heads=3), lambda: cache.plan([a], [1], heads=0),
                lambda: cache.plan([a], [1], new_lengths=[1, 1]), lambda: cache.truncate(a, 1), lambda: cache.truncate(a, -1),
                lambda: cache.fork(9), lambda: cache.free(9)):
        with pytest.raises(ValueError):
            bad()
    assert cache.length(a) == 0 and cache.free_pages == 4
    plan = cache.plan([a], [3], heads=4)
    k, q = torch.zeros(3, 2, 16, dtype=BF), torch.zeros(3, 4, 16, dtype=BF)
    for bad in (lambda: cache_append(cache, 0, k[:2], k, plan), lambda: cache_append(cache, 0, k, k.half(), plan),
                lambda: cache_append(cache, 2, k, k, plan), lambda: cache_append(cache, -1, k, k, plan),
                lambda: cached_attention(k, cache, 0, plan), lambda: cached_attention(q.half(), cache, 0, plan),
                lambda: cached_attention(q, cache, 2, plan), lambda: cached_attention(q, cache, 0, plan, scale=0.0),
                lambda: cached_attention(q, cache, 0, plan, scale=1e39), lambda: cached_attention(q, cache, 0, plan, out=k),
                lambda: cached_attention(q, cache, 0, plan, scale=float("nan")), lambda: cache_read(cache, 2, plan)):
        with pytest.raises(ValueError):
            bad()
    assert cache.plan([a, a], [1, 2], new_lengths=[0, 0]).kv_rows == 6  # read twice, written by none
    for bad in (lambda: cache_append(cache, 0, k.clone().requires_grad_(), k, plan),
                lambda: cached_attention(q.clone().requires_grad_(), cache, 0, plan)):
        with pytest.raises(RuntimeError, match="forward only"):
            bad()


def test_copies_of_pages_on_the_host():
    pool = torch.arange(2 * 6 * 16, dtype=torch.uint8).view(2, 6, 16)
    want = pool.clone()
    want[:, [4, 0]] = want[:, [1, 1]]
    assert copy_pages(pool, [1, 1], [4, 0]) is pool and torch.equal(pool, want)
    for src, dst in (([1], [1]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([6], [0]), ([0], [-1]), ([0], [1, 2])):
        with pytest.raises(ValueError):
            copy_pages(pool, src, dst)
    for bad in (pool[0], pool[:, :, :8], pool.transpose(0, 1), torch.zeros(1, 2, 12, dtype=torch.uint8)):
        with pytest.raises(ValueError):
            copy_pages(bad, [0], [1])
    assert torch.equal(pool, want)


# ---------------------------------------------------------------------------------------------------------------- C ABI

def test_header_and_binding_agree(lib):
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = re.findall(r"^\s*(?:const\s+)?\w+\s*\*?\s*(hf_\w+)\s*\(", text, flags=re.M)
    assert sorted(names) == sorted(_native.CACHE_SIGNATURES)
    for name, (args, _) in _native.CACHE_SIGNATURES.items():
        declared = re.search(name + r"\s*\((.*?)\)", text, flags=re.S).group(1)
        assert len(declared.split(",")) == len(args), name
    kinds = {"int64_t": "q", "int32_t": "i", "float": "f"}
    for name, packer in (("hf_cache_append", _native.CACHE_APPEND_ARGS), ("hf_cache_read", _native.CACHE_READ_ARGS),
                         ("hf_cached_attention", _native.CACHED_ATTENTION_ARGS), ("hf_copy_pages", _native.COPY_PAGES_ARGS),
                         ("hf_residual_norm", _native.RESIDUAL_NORM_ARGS)):
        body = re.search(r"typedef struct \{([^}]*)\} " + name + "_args;", text).group(1)
        fields = [" ".join(p.split()) for p in body.split(";")[:-1]]
        assert packer.format == "@" + "".join(kinds.get(f.rsplit(" ", 1)[0], "P") for f in fields), name
        assert packer.size % struct.calcsize("P") == 0
        assert getattr(lib, name)(None) == -1


def cache_plan(lib, q, kv, new, pages, heads=2, kv_heads=1, D=64, causal=0, page=64, pool=100, cus=256):
    arrays = [(ctypes.c_int64 * max(len(n), 1))(*n) for n in (q, kv, new)]
    table = (ctypes.c_int32 * max(len(pages), 1))(*pages)
    args = (*arrays, len(q), table, pool, page, heads, kv_heads, D, causal, cus)
    n = lib.hf_cache_plan(*args, None, 0)
    if n < 0:
        return n
    buf = ctypes.create_string_buffer(n)
    assert lib.hf_cache_plan(*args, buf, n - 1) == -5
    assert lib.hf_cache_plan(*args, buf, n) == n
    return buf


def test_planner_refuses(lib):
    assert lib.hf_cache_page_bytes(8, 128, 64) == 64 * 8 * 136
    assert lib.hf_cache_page_bytes(1, 96, 32) == 32 * 2 * (48 + 4)
    for args, status in (((0, 128, 64), -1), ((1, 128, 48), -1), ((1, 72, 64), -3), ((1, 144, 64), -5), ((70000, 64, 64), -5)):
        assert lib.hf_cache_page_bytes(*args) == status
    bad = lambda **kw: cache_plan(lib, **({"q": [1], "kv": [70], "new": [1], "pages": [0, 99]} | kw))
    assert isinstance(bad(), ctypes.Array)
    assert bad(pages=[0, 100]) == bad(pages=[-1, 0]) == -1  # pages outside of the pool
    assert bad(new=[71]) == bad(new=[-1]) == bad(q=[-1]) == bad(kv=[-1]) == bad(heads=0) == bad(heads=3, kv_heads=2) == -1
    assert bad(page=16) == bad(cus=65537) == bad(pool=-1) == -1
    assert bad(D=72) == -3 and bad(D=144) == bad(q=[1 << 31]) == bad(pool=1 << 25) == -5
    plan = bad()
    n = len(plan.raw)
    assert lib.hf_cache_ws_bytes(plan, n) >= 0 and lib.hf_cache_ws_bytes(plan, n - 1) == lib.hf_cache_ws_bytes(None, 0) == -1


def test_argument_checks_reject_before_launching(lib):
    fake, odd = 1 << 20, (1 << 20) + 2
    plan = cache_plan(lib, [1, 200], [7000, 80], [1, 3], list(range(110 + 2)), pool=200)
    n, host = len(plan.raw), ctypes.addressof(plan)

    def append(k=fake, token=64, cache=fake, plan=host, dev=fake, size=n, dtype=0):
        return lib.hf_cache_append(_native.CACHE_APPEND_ARGS.pack(k, token, 64, fake, 64, 64, cache, plan, dev, size, dtype, 0))

    assert append(k=0) == append(cache=0) == append(plan=0) == append(dev=0) == append(size=n - 1) == append(dtype=2) == -1
    assert append(token=-8) == -1 and append(k=odd) == append(token=60) == append(cache=odd) == append(dev=odd) == -3

    def read(cache=fake, k=fake, plan=host, dev=fake, size=n, dtype=0):
        return lib.hf_cache_read(_native.CACHE_READ_ARGS.pack(cache, k, fake, plan, dev, size, dtype, 0))

    assert read(cache=0) == read(k=0) == read(plan=0) == read(dev=0) == read(size=n + 1) == read(dtype=-1) == -1
    assert read(cache=odd) == read(k=odd) == read(dev=odd) == -3
    need = lib.hf_cache_ws_bytes(host, n)
    assert need > 0

    def attend(q=fake, token=128, cache=fake, out=fake, scale=0.1, plan=host, dev=fake, size=n, ws=fake, ws_bytes=need,
               dtype=0):
        return lib.hf_cached_attention(_native.CACHED_ATTENTION_ARGS.pack(q, token, 64, cache, out, 128, 64, scale, plan, dev,
                                                                          size, ws, ws_bytes, dtype, 0))

    assert attend(q=0) == attend(cache=0) == attend(out=0) == attend(dev=0) == attend(plan=0) == attend(size=n - 1) == -1
    assert attend(scale=0.0) == attend(scale=float("inf")) == attend(scale=float("nan")) == attend(dtype=3) == -1
    assert attend(ws=0) == attend(ws_bytes=need - 1) == attend(token=-8) == -1
    assert attend(q=odd) == attend(out=odd) == attend(token=130) == attend(ws=odd) == attend(dev=odd) == -3
    empty = cache_plan(lib, [0], [5], [0], [3])
    assert attend(q=0, out=0, plan=ctypes.addressof(empty), size=len(empty.raw)) == 0

    def moves(src, dst, pool=fake, layers=2, layer=1600, pages=100, size=16):
        a, b = ((ctypes.c_int32 * max(len(x), 1))(*x) for x in (src, dst))
        return lib.hf_copy_pages(_native.COPY_PAGES_ARGS.pack(pool, layers, layer, pages, size, ctypes.addressof(a),
                                                              ctypes.addressof(b), len(src), 0))

    assert moves([], []) == moves([1], [2], layers=0) == 0
    assert moves([1], [1]) == moves([1, 2], [3, 3]) == moves([1, 2], [2, 5]) == moves([100], [0]) == moves([0], [-1]) == -1
    assert moves([1], [2], pool=0) == moves([1], [2], layer=1584) == moves([1], [2], layers=-1) == -1
    assert moves([1], [2], size=24) == moves([1], [2], pool=odd) == moves([1], [2], layer=1608) == -3
    assert moves([1], [2], layers=65536) == -5

    names = ("x ldx y ldy r ldr n ldn gate ldg scale lds shift ldh pw w group groups T C post norm per_row wide f32 dtype "
             "residual eps stream").split()
    good = dict(zip(names, [fake, 64, fake, 64, fake, 64, fake, 64, fake, 64, 0, 0, 0, 0, 0, 0, fake, 3, 5, 64, 0, 1, 0, 0, 0, 0,
                            1.0, 1e-6, 0]))

    def norm(**kw):
        return lib.hf_residual_norm(_native.RESIDUAL_NORM_ARGS.pack(*(good | kw).values()))

    assert norm(T=0) == norm(C=0) == 0
    for kw in (dict(x=0), dict(r=0), dict(y=0, n=0), dict(T=-1), dict(post=3), dict(norm=-1), dict(dtype=2), dict(eps=-1.0),
               dict(eps=float("nan")), dict(residual=float("inf")), dict(groups=0), dict(group=0, per_row=1), dict(ldr=56),
               dict(ldn=56), dict(ldx=-8)):
        assert norm(**kw) == -1, kw
    for kw in (dict(C=60), dict(x=odd), dict(gate=odd), dict(ldy=65), dict(ldg=4), dict(w=odd)):
        assert norm(**kw) == -3, kw
    assert norm(C=16392) == norm(T=1 << 31) == -5


def parts(raw):
    """A plan's header fields and its lists."""
    magic, heads, kv_heads, D, causal, page, items, joins = struct.unpack_from("8i", raw, 0)
    _, slots, *_ = struct.unpack_from("6q", raw, 32)
    reads, writes, wides, join_rows = struct.unpack_from("4i", raw, 80)
    at = dict(zip("items joins tables reads writes wides attention attention_bytes".split(), struct.unpack_from("8q", raw, 96)))
    grid = lambda name, n, width: np.frombuffer(raw, np.int32, n * width, at[name]).reshape(n, width)
    rows, = struct.unpack_from("i", raw, 168)
    return {"rows": 16 * rows, "slots": slots, "join_rows": join_rows, "items": grid("items", items, 16), "joins": grid("joins", joins, 8),
            "reads": grid("reads", reads, 4), "writes": grid("writes", writes, 4), "wides": grid("wides", wides, 4),
            "tables": np.frombuffer(raw, np.int32, (at["reads"] - at["tables"]) // 4, at["tables"]),
            "attention": raw[at["attention"]:at["attention"] + at["attention_bytes"]]}


@pytest.mark.parametrize("cus", [1, 256])
@pytest.mark.parametrize("q,kv,new,heads,kv_heads,causal,page", [
    ([1] * 16, [8191, 4096, 733, 1, 16384, 2500, 6001, 127, 9999, 3000, 512, 7777, 64, 12001, 1025, 5000], [1] * 16, 32, 8, 1, 64),
    ([5, 0, 300, 1, 7], [5, 9, 300, 40000, 0], [5, 0, 20, 1, 0], 8, 2, 1, 32), ([1], [131072], [0], 64, 8, 0, 256),
    ([], [], [], 2, 1, 0, 64), ([1, 800, 0, 90, 700], [50000, 60000, 5, 300, 9000], [1, 3, 0, 0, 700], 4, 2, 1, 128),
    ([1, 800, 0, 90], [70, 60000, 5, 300], [1, 3, 0, 0], 4, 2, 1, 128), ([3, 65], [0, 0], [0, 0], 2, 2, 1, 64), ([40], [3], [3], 1, 1, 1, 128), ([900], [1000], [900], 1, 1, 0, 64)])
def test_plan_covers_every_row_key_and_token_once(lib, q, kv, new, heads, kv_heads, causal, page, cus):
    counts = [-(-n // page) for n in kv]
    order = list(range(sum(counts)))
    random.Random(1).shuffle(order)
    plan = cache_plan(lib, q, kv, new, order, heads, kv_heads, 64, causal, page, max(len(order), 1), cus)
    p = parts(plan.raw)
    group = heads // kv_heads
    # segments: each token in its page and row
    tables = [order[sum(counts[:i]):sum(counts[:i + 1])] for i in range(len(kv))]
    assert p["tables"].tolist()[:len(order)] == order

    def rows(segments):
        return sorted((row0 + i, page_, first + i) for page_, first, n, row0 in segments.tolist() for i in range(n))

    def want(spans):
        return [(row, tables[b][t // page], t % page) for row, (b, t) in enumerate(
            (b, t) for b, (lo, hi) in spans for t in range(lo, hi))]

    assert rows(p["reads"]) == want([(b, (0, n)) for b, n in enumerate(kv)])
    assert rows(p["writes"]) == want([(b, (n - m, n)) for b, (n, m) in enumerate(zip(kv, new))])
    assert bool(p["attention"]) == (60000 in kv)
    wide = [b for b in range(len(q)) if p["attention"] and q[b] * group >= (320 if 50000 in kv else 1)]
    assert rows(p["wides"]) == want([(b, (0, kv[b])) for b in wide])
    # items: every row of the sequences that are not expanded, over every key that its last row sees, once
    seen = {}
    q0 = [sum(q[:b]) for b in range(len(q))]
    for item in p["items"].tolist():
        a, nq, nk, row0, lo, hi, head, slot, table0 = item[:9]
        b = next(b for b in range(len(q)) if q0[b] == a and q[b] == nq and sum(counts[:b]) == table0 and kv[b] == nk and q[b])
        assert b not in wide and lo % 32 == 0 and 0 <= lo <= hi <= nk and (hi % 32 == 0 or hi <= nk)
        seen.setdefault((b, head, row0), []).append((lo, hi, slot))
        assert all(item[9 + i] == tables[b][key // page] for i, key in enumerate(range(lo, min(hi, lo + 128), 32)))
    slots = []
    for b in range(len(q)):
        if b in wide:
            continue
        for head in range(kv_heads):
            for row0 in range(0, q[b] * group, p["rows"]):
                spans = sorted(seen.pop((b, head, row0)))
                last = min(row0 + p["rows"], q[b] * group) - 1
                hi = min(max(last // group + kv[b] - q[b] + 1, 0), kv[b]) if causal else kv[b]
                assert spans[0][0] == 0 and spans[-1][1] == hi and all(x[1] == y[0] for x, y in zip(spans, spans[1:]))
                assert (spans[0][2] < 0) == (len(spans) == 1)
                slots += [s for *_, s in spans if s >= 0]
    assert not seen and sorted(slots) == list(range(p["slots"]))
    joined = [s for *_, slot0, n, rows_ in p["joins"].tolist() for s in range(slot0, slot0 + n)]
    assert sorted(joined) == sorted(slots)
    assert all(1 <= j[7] <= p["join_rows"] <= 32 for j in p["joins"].tolist())
    # the expanded sequences' attention: their queries where they lie, their keys one behind the other
    if wide:
        n, = struct.unpack_from("i", p["attention"], 20)
        items = np.frombuffer(p["attention"], np.int32, n * 12, 128).reshape(n, 12).tolist()
        starts = {(q0[b], q[b], sum(kv[w] for w in wide if w < b), kv[b]) for b in wide}
        assert {tuple(i[:4]) for i in items} == starts


def expanded(raw):
    """The items and joins of a plan's attention over expanded keys, and whether the join for few shares takes them."""
    raw = parts(raw)["attention"]
    items, joins, few = struct.unpack_from("3i", raw, 20)
    slots, = struct.unpack_from("q", raw, 40)
    assert len(raw) == 128 + 48 * items + 32 * joins
    return (np.frombuffer(raw, np.int32, items * 12, 128).reshape(-1, 12).tolist(),
            np.frombuffer(raw, np.int32, joins * 8, 128 + 48 * items).reshape(-1, 8).tolist(), slots, bool(few))


@pytest.mark.parametrize("q,kv,heads,kv_heads,D,causal,few,unequal", [
    ([4860], [37710], 7, 7, 128, 0, True, True), ([4860], [40000], 7, 7, 128, 0, True, True),
    ([4700], [37710], 7, 7, 128, 0, False, True), ([512, 300, 61, 1], [4096, 8191, 733, 2500], 32, 8, 128, 1, True, True),
    ([2000], [4000], 16, 16, 128, 0, True, False), ([400], [90000], 2, 1, 128, 1, False, False),
    ([2300], [5000], 16, 16, 80, 1, True, True), ([700, 650, 900], [3000, 5000, 9000], 16, 8, 96, 1, True, True),
    ([1500, 0, 320], [6001, 70, 0], 24, 24, 64, 0, True, True), ([800, 5], [16000, 9], 8, 8, 128, 1, True, False)])
def test_expanded_parts_cover_each_tile_of_rows_once(lib, q, kv, heads, kv_heads, D, causal, few, unequal):
    """Parts of a tile of 128 rows take all keys that its last row sees once, from one key tile's start to another's, each with
    a share of its own that one join reads; the cuts and the join are the ones that the case stands for."""
    counts = [-(-n // 64) for n in kv]
    group = heads // kv_heads
    for cus in (256, 7):
        raw = cache_plan(lib, q, kv, [0] * len(q), list(range(sum(counts))), heads, kv_heads, D, causal, 64, sum(counts), cus).raw
        items, joins, slots, quick = expanded(raw)
        wide = [b for b in range(len(q)) if any(i[0] == sum(q[:b]) and i[1] == q[b] for i in items) and q[b]]
        assert wide
        want = {}  # (first query, queries, first key, keys, first row, head): keys of the tile
        for i, b in enumerate(wide):
            for head in range(kv_heads):
                for row0 in range(0, q[b] * group, 128):
                    last = min(row0 + 128, q[b] * group) - 1
                    hi = min(max(last // group + kv[b] - q[b] + 1, 0), kv[b]) if causal else kv[b]
                    want[sum(q[:b]), q[b], sum(kv[w] for w in wide[:i]), kv[b], row0, head] = hi
        spans = {}
        for q0, nq, k0, nk, row0, lo, hi, head, slot, *_ in items:
            spans.setdefault((q0, nq, k0, nk, row0, head), []).append((lo, hi, slot))
        assert spans.keys() == want.keys()
        joined = {(q0, nq, k0, nk, row0, head): list(range(slot, slot + n)) for q0, nq, k0, nk, row0, head, slot, n in joins}
        assert len(joined) == len(joins)
        uneven, seen = 0, []
        for tile, cut in spans.items():
            cut.sort()
            assert cut[0][0] == 0 and cut[-1][1] == want[tile] and all(a[1] == b[0] for a, b in zip(cut, cut[1:]))
            assert all(lo % 64 == 0 and (lo < hi or hi == 0) for lo, hi, _ in cut)
            shares = [slot for *_, slot in cut]
            assert sorted(shares) == joined.pop(tile, [-1]) and (len(cut) > 1) == (shares[0] >= 0)
            seen += [s for s in shares if s >= 0]
            sizes = [hi - lo for lo, hi, _ in cut]
            uneven += max(sizes) - min(sizes) > 128  # equal cuts differ by a key tile and the end of the last
        assert not joined and sorted(seen) == list(range(slots))
        most = max([n for *_, n in joins], default=0)
        assert quick == (4 * most <= len(joins))
        if cus == 256:
            assert joins and quick == few and (uneven > 0) == unequal


def passes(raw):
    """The passes of a plan's expanded sequences: (first segment, segments, rows, where the plan of its attention lies, bytes)."""
    n, = struct.unpack_from("i", raw, 172)
    at, = struct.unpack_from("q", raw, 176)
    return [struct.unpack_from("2i3q", raw, at + 32 * i) for i in range(n)]


@pytest.mark.parametrize("q,kv,heads,kv_heads,D,sizes", [
    ([200] * 24, [100000] * 24, 32, 8, 128, [1000000, 1000000, 400000]),
    ([200, 0, 200, 700, 200], [1 << 20, 9000, 1, 1200000, (1 << 20) - 1], 32, 8, 128, [1 << 20, 1, 1200000, (1 << 20) - 1]),
    ([4860], [37710], 7, 7, 128, [37710]), ([400, 400], [2500000, 2000000], 16, 4, 64, [2500000, 2000000])])
def test_expanded_sequences_share_a_bounded_workspace(lib, q, kv, heads, kv_heads, D, sizes):
    """Long batches are expanded pass by pass: up to 2^32 bytes of keys and values, or one sequence, at a time."""
    counts = [-(-n // 64) for n in kv]
    pages = list(range(sum(counts)))[::-1]
    plan = cache_plan(lib, q, kv, [0] * len(q), pages, heads, kv_heads, D, 1, 64, sum(counts))
    found = passes(plan.raw)
    assert [rows for _, _, rows, _, _ in found] == sizes
    assert lib.hf_cache_ws_bytes(plan, len(plan.raw)) <= max(1 << 32, 4 * max(sizes) * kv_heads * D) + (100 << 20)
    segments = parts(plan.raw)["wides"].tolist()
    b = segment = 0
    for first, count, rows, at, size in found:
        assert first == segment
        segment += count
        want, items, row = [], set(), 0  # segments of the pass's sequences, one behind the other, their queries and first keys
        while row < rows:
            if q[b]:  # those without queries are not expanded
                items.add((sum(q[:b]), q[b], row, kv[b]))
                table = pages[sum(counts[:b]):sum(counts[:b + 1])]
                want += [[page, 0, min(64, kv[b] - 64 * i), row + 64 * i] for i, page in enumerate(table)]
                row += kv[b]
            b += 1
        assert row == rows and segments[first:segment] == want
        n, = struct.unpack_from("i", plan.raw, at + 20)
        raw = plan.raw[at:at + size]
        assert {tuple(i[:4]) for i in np.frombuffer(raw, np.int32, n * 12, 128).reshape(n, 12).tolist()} == items
    assert b == len(q) and segment == len(segments)


# ------------------------------------------------------------------------------------------------------- residual norms

@pytest.mark.parametrize("norm,post", [("rms", None), ("layer", "rms"), (None, "layer")])
def test_host_norms(norm, post):
    lens = [3, 0, 5]
    x, y, m = rnd(1, 8, 40).float(), rnd(2, 8, 40).to(BF), rnd(3, 3, 3, 40).to(BF)
    w = (1 + 0.1 * rnd(4, 40)).to(BF)
    rows = RowPlan(lens, device="cpu")
    got = residual_norm(x, y, rows=rows, residual=0.5, gate=m[:, 0], post_norm=post, post_weight=w, norm=norm, weight=w,
                        scale=m[:, 1], shift=m[:, 2])
    r, n = C.residual_norm(x, y, rows.groups.long(), 0.5, m[:, 0], post, w, norm, w, m[:, 1], m[:, 2], 1e-6, BF)
    U.check(got[0], *r)
    U.check(got[1], *n)
    a, b = torch.empty_like(x), torch.empty_like(y)
    again = residual_norm(x, y, rows=rows, residual=0.5, gate=m[:, 0], post_norm=post, post_weight=w, norm=norm, weight=w,
                          scale=m[:, 1], shift=m[:, 2], out=(a, b))
    assert again[0] is a and again[1] is b and torch.equal(a, got[0]) and torch.equal(b, got[1])


def test_refusals_of_the_norms():
    x, y, v = torch.zeros(4, 64, dtype=BF), torch.zeros(4, 64, dtype=BF), torch.zeros(64, dtype=BF)
    rows = RowPlan([1, 3], device="cpu")
    for bad in (
        lambda: residual_norm(x[0]), lambda: residual_norm(x, y[:3]), lambda: residual_norm(x[:, :60], y[:, :60]),
        lambda: residual_norm(torch.zeros(1, 16392, dtype=BF)), lambda: residual_norm(x[:, :0]),
        lambda: residual_norm(x.half(), y), lambda: residual_norm(x, y.float()), lambda: residual_norm(x.double(), y),
        lambda: residual_norm(x, y, dtype=HF), lambda: residual_norm(x, y, norm="batch"),
        lambda: residual_norm(x, y, post_norm="batch"), lambda: residual_norm(x, gate=v), lambda: residual_norm(x, residual=2.0),
        lambda: residual_norm(x, post_norm="rms"), lambda: residual_norm(x, norm=None),
        lambda: residual_norm(x, y, residual=float("nan")), lambda: residual_norm(x, y, residual=1e39),
        lambda: residual_norm(x, y, eps=-1.0), lambda: residual_norm(x, y, eps=float("nan")),
        lambda: residual_norm(x, y, rows=RowPlan([3], device="cpu")), lambda: residual_norm(x, y, gate=v[:63]),
        lambda: residual_norm(x, y, rows=rows, gate=v.expand(4, 64)), lambda: residual_norm(x, y, gate=v.expand(2, 64)),
        lambda: residual_norm(x, y, weight=v[None]), lambda: residual_norm(x, y, weight=v.half()),
        lambda: residual_norm(x, y, out=(x, None)),
        lambda: residual_norm(x, y, norm=None, out=(x, y)), lambda: residual_norm(x, y, out=(x, y.float())),
        lambda: residual_norm(x, y, out=(x[:3], y)), lambda: residual_norm(x, out=(x, y)),
        lambda: residual_norm(x, y, out=(x, x)), lambda: RowPlan([-1], device="cpu"),
    ):
        with pytest.raises(ValueError):
            bad()
    for t in ((x.clone().requires_grad_(), y), (x, y.clone().requires_grad_())):
        with pytest.raises(RuntimeError, match="forward only"):
            residual_norm(*t)
    with torch.no_grad():
        residual_norm(x.clone().requires_grad_(), y)

"""The 4-bit cache on the GPU: pages written and read back bit by bit, attention over them against 64 bits, copies of pages."""

from __future__ import annotations

import copy
import threading

import pytest
import torch

import block_utils as U
import cache_utils as C
from hyperflow_h3_flash_amd import KVCache, cache_append, cache_read, cached_attention, copy_pages
from test_cache import expanded, passes

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _name(request):
    print(f"case {request.node.name}", flush=True)


def rnd(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).cuda()


def keys(seed, rows, heads, D, dtype, spread=0):
    """Values whose magnitudes span 2^+-spread by group."""
    x = rnd(seed, rows, heads, D)
    if spread:
        e = torch.randint(-spread, spread + 1, (rows, heads, -(-D // 32)), generator=torch.Generator().manual_seed(seed + 1))
        x = torch.ldexp(x, e.cuda().repeat_interleave(32, -1)[..., :D])
    return x.to(dtype)


def filled(kv, hk, D, dtype=BF, page=64, layers=1, layer=0, seed=0, steps=2, spare=0, fill=None, k=None, v=None):
    """A cache that holds the sequences, written in several steps so that their pages lie among one another."""
    pages = sum(-(-n // page) for n in kv) + spare
    cache = KVCache(layers, hk, D, pages, page_size=page, dtype=dtype)
    if fill is not None:
        cache.data.fill_(fill)
    k = keys(seed + 1, sum(kv), hk, D, dtype) if k is None else k
    v = (keys(seed + 3, sum(kv), hk, D, torch.float32) + 0.5).to(dtype) if v is None else v
    requests = [cache.new() for _ in kv]
    at = [0] * len(kv)
    for i in range(steps):
        new = [n * (i + 1) // steps - n * i // steps for n in kv]
        take = torch.cat([torch.arange(a, a + b) + s for a, b, s in zip(at, new, [sum(kv[:j]) for j in range(len(kv))])]
                         or [torch.arange(0)]).cuda()
        cache_append(cache, layer, k[take], v[take], cache.plan(requests, new))
        at = [a + b for a, b in zip(at, new)]
    return cache, requests, k, v


# ------------------------------------------------------------------------------------------------------ write and read

@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [16, 32, 48, 64, 80, 96, 112, 128])
@pytest.mark.parametrize("page", [32, 256])
def test_pages_are_the_hosts_and_read_exactly(D, dtype, page):
    kv, hk = [1, page, page + 1, 0, 3 * page - 1, 7], 3
    k, v = (keys(s, sum(kv), hk, D, dtype, spread=9) for s in (1, 5))
    k[3, 1, :16], v[5, 0, -16:] = 0.0, 0.0
    cache, requests, _, _ = filled(kv, hk, D, dtype, page, fill=0xA5, k=k, v=v, spare=2)
    host = KVCache(1, hk, D, cache.pages, page_size=page, dtype=dtype, device="cpu")
    host.data.fill_(0xA5)
    mine = [host.new() for _ in kv]
    at = [0] * len(kv)
    for i in range(2):
        new = [n * (i + 1) // 2 - n * i // 2 for n in kv]
        take = torch.cat([torch.arange(a, a + b) + sum(kv[:j]) for j, (a, b) in enumerate(zip(at, new))])
        cache_append(host, 0, k.cpu()[take], v.cpu()[take], host.plan(mine, new))
        at = [a + b for a, b in zip(at, new)]
    assert torch.equal(cache.data.cpu(), host.data)  # with what no token wrote left as it was
    got = cache_read(cache, 0, cache.plan(requests, [0] * len(kv)))
    for a, x in zip(got, (k, v)):
        assert a.dtype is dtype and torch.equal(a.double(), C.held(x))


@pytest.mark.parametrize("dtype", [BF, HF])
def test_every_value_of_the_type(dtype):
    """Each 16-bit value as the largest of a group whose others are its fractions."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype).cuda()
    x = torch.zeros(65536, 1, 32, dtype=dtype, device="cuda")
    x[:, 0, 0] = bits
    x[:, 0, 1:] = (bits.float()[:, None] * torch.linspace(-1, 1, 31, device="cuda")).to(dtype)
    cache, requests, _, _ = filled([65536], 1, 32, dtype, k=x, v=x.flip(0), steps=1)
    k, v = cache_read(cache, 0, cache.plan(requests, [0]))
    want = C.held(x)
    for got, ref in ((k, want), (v, want.flip(0))):
        assert torch.equal(got.isnan(), ref.isnan())
        assert torch.equal(got.double().nan_to_num(7.0), ref.nan_to_num(7.0))
    fine = ~want.isnan()
    # half a step at most: one of the scale's units between 4 and 6, except where the scale is at its limit
    top = 6 * 2.0 ** C.LIMITS[dtype][1]
    off = (want - x.double()).abs()[fine]
    assert (off <= torch.maximum(x.double().abs().amax(-1, keepdim=True).expand_as(x)[fine] / 3.5,
                                 torch.tensor(2.0 ** C.LIMITS[dtype][0])))[x.double().abs()[fine] <= top].all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_a_group_that_is_not_finite_reads_as_nan_and_no_other(bad):
    k, v = keys(1, 70, 2, 80, BF), keys(2, 70, 2, 80, BF)
    k[5, 1, 40] = bad
    v[69, 0, 79] = bad
    cache, requests, _, _ = filled([70], 2, 80, k=k, v=v)
    got = cache_read(cache, 0, cache.plan(requests, [0]))
    nan = torch.zeros(2, 70, 2, 80, dtype=torch.bool, device="cuda")
    nan[0, 5, 1, 32:64] = nan[1, 69, 0, 64:80] = True
    for i, x in enumerate((k, v)):
        assert torch.equal(got[i].isnan(), nan[i])
        assert torch.equal(got[i].double().nan_to_num(9.0), C.held(x).nan_to_num(9.0))


def test_strides_of_projections_and_heads_first():
    wide = rnd(1, 300, 12, 64).to(BF)
    k, v = wide[:, 4:8], rnd(2, 4, 300, 64).to(BF).transpose(0, 1)
    odd = rnd(3, 300, 4, 65).to(BF)[..., 1:]  # not on a 16-byte boundary
    for a, b in ((k, v), (v, odd)):
        cache, requests = KVCache(1, 4, 64, 5), None
        requests = [cache.new()]
        cache_append(cache, 0, a, b, cache.plan(requests, [300]))
        got = cache_read(cache, 0, cache.plan(requests, [0]))
        assert torch.equal(got[0].double(), C.held(a)) and torch.equal(got[1].double(), C.held(b))


# ----------------------------------------------------------------------------------------------------------- attention

def run_attention(q_lens, kv_lens, hq, hk, D, dtype=BF, causal=False, scale=None, page=64, seed=0, spread=1.0, fill=0xFF):
    """Pages hold 0xFF (NaN scales) where no token is."""
    cache, requests, k, v = filled(kv_lens, hk, D, dtype, page, fill=fill, seed=seed)
    q = (spread * rnd(seed + 9, sum(q_lens), hq, D)).to(dtype)
    plan = cache.plan(requests, q_lens, new_lengths=[0] * len(kv_lens), heads=hq, causal=causal)
    got = cached_attention(q, cache, 0, plan, scale=scale)
    ref, bound = C.attention(q, k, v, q_lens, kv_lens, causal, D ** -0.5 if scale is None else scale)
    U.check(got, ref, bound, f"{q_lens} {kv_lens} {hq}/{hk} x {D}")
    return cache, plan, q, k, v, got


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 160, 257])
def test_lengths_around_blocks_and_pages(n, causal):
    for q in (1, min(n, 5)):
        run_attention([q], [n], 4, 2, 128, causal=causal, page=32 if n % 2 else 64, seed=n)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("D", [16, 32, 48, 64, 80, 96, 112, 128])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_head_widths_and_types(D, dtype, causal):
    run_attention([3, 1, 40], [200, 77, 40], 6, 3, D, dtype, causal, seed=D)


@pytest.mark.parametrize("hq,hk", [(1, 1), (5, 1), (8, 2), (7, 7), (40, 1), (16, 1), (33, 1), (64, 2), (100, 1)])
def test_head_groups(hq, hk):
    run_attention([1, 2], [300, 90], hq, hk, 64, causal=True)


@pytest.mark.parametrize("page", [32, 64, 128, 256])
def test_page_sizes(page):
    run_attention([1, 4, 2], [1000, 65, 513], 8, 2, 128, causal=True, page=page)


@pytest.mark.parametrize("q,kv", [(1, 20000), (5, 9000), (33, 2049), (70, 3000)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_few_rows_over_many_keys_are_cut_and_joined(q, kv, dtype):
    run_attention([q], [kv], 2, 1, 128, dtype, causal=True)


def test_few_and_many_rows_in_one_batch():
    run_attention([1, 300, 0, 7, 129], [700, 300, 40, 1200, 400], 8, 2, 96, causal=True)
    run_attention([300, 1, 200], [100, 9, 0], 4, 4, 64, causal=False)


@pytest.mark.parametrize("dtype,D,causal", [(BF, 128, True), (HF, 64, False), (HF, 96, True)])
def test_expanded_sequences_beside_others(dtype, D, causal):
    """Many rows over many keys go through a workspace of 16-bit keys and values, few rows of the same batch do not."""
    for one in (300, 50000):
        cache, plan, *_ = run_attention([2, 360, 0, 40], [one, 100001, 5, 900], 4, 2, D, dtype, causal)
        rows = 100001 + (0 if one > 300 else 300 + 5 + 900)
        assert 0 <= plan.ws_bytes - 2 * rows * 2 * D * 2 < 60 << 20  # shares come to less


CUTS = [  # (..., the join for few shares, cuts of unequal length): test_cache.py holds the plans to them
    ([2300], [5000], 16, 16, 80, True, True, True), ([1500, 0, 320], [6001, 70, 0], 24, 24, 64, False, True, True),
    ([2000], [4000], 16, 16, 128, False, True, False), ([700, 650, 900], [3000, 5000, 9000], 16, 8, 96, True, True, True),
    ([4700], [37710], 7, 7, 128, False, False, True), ([400], [90000], 2, 1, 128, True, False, False)]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("q,kv,hq,hk,D,causal,few,unequal", CUTS)
def test_expanded_cuts_and_both_joins(q, kv, hq, hk, D, causal, few, unequal, dtype):
    _, plan, *_ = run_attention(q, kv, hq, hk, D, dtype, causal)
    items, joins, _, quick = expanded(plan.data.host.numpy().tobytes())
    spans = {}
    for q0, _, _, _, row0, lo, hi, head, *_ in items:
        spans.setdefault((q0, row0, head), []).append(hi - lo)
    assert joins and quick == few and any(max(n) - min(n) > 128 for n in spans.values()) == unequal


def test_sequences_expanded_pass_by_pass():
    """More keys than a pass takes: the workspace is the longest pass's, results are those of the sequences alone."""
    q_lens, kv_lens, hq, hk, D = [170, 200, 3, 180], [500003, 500000, 900, 120001], 32, 8, 128
    gen = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn(sum(kv_lens), hk, D, generator=gen, device="cuda").to(BF) for _ in range(2))
    cache, requests, _, _ = filled(kv_lens, hk, D, k=k, v=v)
    q = rnd(2, sum(q_lens), hq, D).to(BF)
    plan = cache.plan(requests, q_lens, new_lengths=[0] * 4, heads=hq, causal=True)
    assert len(passes(plan.data.host.numpy().tobytes())) == 2 and plan.ws_bytes < (1 << 32) + (100 << 20)
    got = cached_attention(q, cache, 0, plan)
    held_k, held_v = cache_read(cache, 0, plan)
    ref, bound = U.attention(q, held_k, held_v, q_lens, kv_lens, True, D ** -0.5)
    U.check(got, ref, bound)
    assert torch.equal(cached_attention(q, cache, 0, plan, out=q), got)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_nan_that_some_rows_see_through_unequal_cuts(dtype):
    q_len, kv, heads, D = 2300, 5000, 16, 80
    k, v = keys(1, kv, heads, D, dtype), keys(2, kv, heads, D, dtype)
    fine = v.clone()
    v[kv - 51, 3, 70] = float("nan")  # seen by the last 51 queries
    v[100, 5, 10] = float("inf")  # by all
    k[kv - 2, 7, 3] = float("nan")  # by the last two
    nan = torch.zeros(q_len, heads, D, dtype=torch.bool, device="cuda")
    nan[-51:, 3, 64:80] = nan[:, 5, :32] = nan[-2:, 7] = True
    fine[kv - 51, 3, 64:80] = fine[100, 5, :32] = 0
    kk = k.clone()
    kk[kv - 2, 7, :32] = 0
    cache, requests, _, _ = filled([kv], heads, D, dtype, k=k, v=v)
    q = rnd(3, q_len, heads, D).to(dtype)
    plan = cache.plan(requests, [q_len], new_lengths=[0], heads=heads, causal=True)
    assert expanded(plan.data.host.numpy().tobytes())[3]
    got = cached_attention(q, cache, 0, plan)
    assert torch.equal(got.isnan(), nan)
    ref, bound = C.attention(q, kk, fine, [q_len], [kv], True, D ** -0.5)
    U.check(torch.where(nan, 0.0, got.double()), torch.where(nan, 0.0, ref), bound)


@pytest.mark.parametrize("causal", [False, True])
def test_queries_without_keys_and_caches_without_queries(causal):
    for q, kv in (([5, 90], [0, 0]), ([9, 200], [3, 5]), ([0, 0], [70, 5]), ([0], [0]), ([], [])):
        *_, got = run_attention(q, kv, 2, 2, 32, causal=causal)
    cache, requests, _, _ = filled([], 2, 32)
    assert cached_attention(rnd(1, 4, 2, 32).to(BF), cache, 0, cache.plan([cache.new()], [4], new_lengths=[0])).eq(0).all()


def test_scale_and_sharp_scores():
    run_attention([1, 9], [500, 300], 4, 2, 64, scale=0.7, spread=4.0, causal=True)
    run_attention([1, 9], [500, 300], 4, 2, 64, HF, scale=3.0, spread=2.0)
    run_attention([2], [300], 4, 2, 64, scale=1e-30)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_rising_maxima_and_a_dominant_key(dtype):
    k = torch.zeros(600, 1, 32, dtype=dtype, device="cuda")
    k[:, 0, 0] = torch.arange(600, device="cuda") / 8  # scores rise block after block
    k[577, 0, 0] = 120
    v = keys(4, 600, 1, 32, dtype)
    cache, requests, k, v = filled([600], 1, 32, dtype, k=k, v=v)
    q = torch.zeros(3, 1, 32, dtype=dtype, device="cuda")
    q[:, 0, 0] = torch.tensor([1.0, -1.0, 0.2])
    plan = cache.plan(requests, [3], new_lengths=[0])
    ref, bound = C.attention(q, k, v, [3], [600], False, 1.0)
    U.check(cached_attention(q, cache, 0, plan, scale=1.0), ref, bound)


@pytest.mark.parametrize("rows,kv", [(3, 200), (130, 200), (400, 90000)])
def test_unseen_nan_stays_out_and_seen_nan_shows(rows, kv):
    """A key or value group that is not finite reaches the rows that see it and no other; on pages and expanded."""
    hq, D = 2, 128
    k, v = keys(1, kv, 1, D, BF), keys(2, kv, 1, D, BF)
    k[kv - 2, 0, 3] = float("inf")  # seen by the last two queries
    v[kv - 1, 0, 70] = float("nan")  # by the last
    v[5, 0, 100] = float("nan")  # by all
    cache, requests, _, _ = filled([kv], 1, D, k=k, v=v)
    q = rnd(3, rows, hq, D).to(BF)
    got = cached_attention(q, cache, 0, cache.plan(requests, [rows], new_lengths=[0], heads=hq, causal=True))
    nan = torch.zeros(got.shape, dtype=torch.bool, device="cuda")
    nan[:, :, 96:128] = True
    nan[-2:] = True
    assert torch.equal(got.isnan(), nan)
    fine = v.clone()
    fine[5, 0, 96:128] = 0
    fine[kv - 1, 0, 64:96] = 0
    kk = k.clone()
    kk[kv - 2, 0, :32] = 0
    ref, bound = C.attention(q, kk, fine, [rows], [kv], True, D ** -0.5)
    U.check(got[:-2, :, :96], ref[:-2, :, :96], bound[:-2, :, :96])


def test_all_keys_nan():
    k = torch.full((40, 1, 32), float("nan"), dtype=BF, device="cuda")
    cache, requests, _, _ = filled([40], 1, 32, k=k, v=keys(1, 40, 1, 32, BF))
    assert cached_attention(rnd(2, 2, 1, 32).to(BF), cache, 0, cache.plan(requests, [2], new_lengths=[0])).isnan().all()
    k = keys(3, 400, 1, 32, BF)
    k[64:96] = float("nan")  # one wave's whole block
    cache, requests, _, _ = filled([400], 1, 32, k=k, v=keys(1, 400, 1, 32, BF))
    got = cached_attention(rnd(2, 400, 1, 32).to(BF)[:10], cache, 0, cache.plan(requests, [10], new_lengths=[0]))
    assert got.isnan().all()


@pytest.mark.parametrize("dtype", [BF, HF])
def test_ends_of_the_type(dtype):
    top = torch.finfo(dtype).max
    v = torch.full((70, 1, 32), top, dtype=dtype, device="cuda")
    k = torch.full((70, 1, 32), torch.finfo(dtype).smallest_normal, dtype=dtype, device="cuda")
    cache, requests, _, _ = filled([70], 1, 32, dtype, k=k, v=v)
    got = cache_read(cache, 0, cache.plan(requests, [0]))
    assert torch.equal(got[0].double(), C.held(k)) and torch.equal(got[1].double(), C.held(v)) and got[1].isfinite().all()
    q = rnd(1, 1, 1, 32).to(dtype)
    out = cached_attention(q, cache, 0, cache.plan(requests, [1], new_lengths=[0]))
    # 70 equal values: the sum of 70 of bfloat16's largest passes float32 (as in packed attention); float16's does not.
    if dtype is HF:
        U.check(out, C.held(v)[:1], C.held(v)[:1] * 2 * 2.0 ** -11)


@pytest.mark.parametrize("rows", [1, 40])
def test_values_up_to_the_stated_range_of_bfloat16(rows):
    """Values times 256 times the number of keys may reach float32's range; equal values past it overflow their sum."""
    n = 70
    inside = 6.0 * 2.0 ** 111  # times 256 * 70: 2.8e38
    assert inside * 256 * n < torch.finfo(torch.float32).max < 2 * inside * 256 * n
    k, q = keys(1, n, 1, 32, BF), rnd(2, rows, 1, 32).to(BF)
    for value, finite in ((inside, True), (-inside, True), (torch.finfo(BF).max, False)):
        v = torch.full((n, 1, 32), value, dtype=BF, device="cuda")
        v[:, 0, 1] *= 0.25  # another level of the same scale
        cache, requests, _, _ = filled([n], 1, 32, k=k, v=v)
        got = cached_attention(q, cache, 0, cache.plan(requests, [rows], new_lengths=[0]))
        ref, bound = C.attention(q, k, v, [rows], [n], False, 32 ** -0.5)
        if finite:
            U.check(got, ref, bound)
        else:  # 70 weights of up to 2^8, of which one is 1 or more: a sum of at least the value, up to infinity, never NaN
            assert not got.isnan().any() and (got.double() >= (ref - bound).clamp_max(torch.finfo(BF).max)).all()


@pytest.mark.parametrize("dtype", [BF, HF])
def test_no_farther_from_packed_attention_than_both_may_be_off(dtype):
    from hyperflow_h3_flash_amd import AttentionPlan, packed_attention
    q_lens, kv_lens = [2, 130, 1, 40], [700, 300, 64, 0]
    cache, plan, q, *_, got = run_attention(q_lens, kv_lens, 8, 4, 128, dtype, causal=True)
    k, v = cache_read(cache, 0, plan)
    other = packed_attention(q, k, v, AttentionPlan(q_lens, kv_lens, heads=8, kv_heads=4, head_dim=128, causal=True))
    ref, bound = U.attention(q, k, v, q_lens, kv_lens, True, 128 ** -0.5)
    U.check(got, ref, bound)
    U.check(other, ref, bound)
    assert ((got.double() - other.double()).abs() <= 2 * bound).all()


def test_out_in_place_and_strided():
    cache, plan, q, k, v, want = run_attention([3, 200], [300, 200], 4, 2, 64, causal=True)
    for out in (torch.empty_like(q), torch.zeros(203, 9, 64, dtype=BF, device="cuda")[:, 2:6],
                torch.zeros(4, 203, 64, dtype=BF, device="cuda").transpose(0, 1)):
        assert cached_attention(q, cache, 0, plan, out=out) is out and torch.equal(out, want)
    wide = torch.zeros(203, 8, 64, dtype=BF, device="cuda")
    wide[:, 1:5] = q
    shifted = wide[:, 2:6]
    assert torch.equal(cached_attention(wide[:, 1:5], cache, 0, plan, out=shifted), want)
    q2 = q.clone()
    version = q2._version
    assert cached_attention(q2, cache, 0, plan, out=q2) is q2 and torch.equal(q2, want) and q2._version > version
    version = cache.data._version
    cache_append(cache, 0, k[:0], v[:0], cache.plan([0], [0]))
    assert cache.data._version == version


def test_layers_past_32_bits():
    """The last of several layers, whose pages lie more than 4 GiB behind the pool's start, and a page far into a layer."""
    cache = KVCache(3, 8, 128, 30000, page_size=64)  # 2 GiB a layer
    assert cache.data[0].numel() > 2 ** 31 - 2 ** 27 and cache.data.numel() > 2 ** 32
    other = cache.new()
    cache.plan([other], [64 * 29990])
    request = cache.new()
    k, v = keys(1, 300, 8, 128, BF), keys(2, 300, 8, 128, BF)
    plan = cache.plan([request], [300], heads=8, causal=True)
    assert min(cache.table(request)) >= 29990
    cache_append(cache, 2, k, v, plan)
    got = cache_read(cache, 2, plan)
    assert torch.equal(got[0].double(), C.held(k)) and torch.equal(got[1].double(), C.held(v))
    q = rnd(3, 300, 8, 128).to(BF)
    ref, bound = C.attention(q, k, v, [300], [300], True, 128 ** -0.5)
    U.check(cached_attention(q, cache, 2, plan), ref, bound)
    one = cache.plan([request], [1], new_lengths=[0], causal=True)
    U.check(cached_attention(q[-1:], cache, 2, one), ref[-1:], bound[-1:])
    page = cache.data[2, cache.table(request)[0]].clone()
    copy_pages(cache.data, [cache.table(request)[0]], [29999])
    assert torch.equal(cache.data[2, 29999], page) and cache.data[1, 29999].eq(0).all()


def test_same_bits_every_time_and_rows_alone():
    cache, plan, q, k, v, want = run_attention([1, 4, 150, 2], [5000, 800, 700, 64], 8, 2, 128, causal=True)
    for _ in range(5):
        assert torch.equal(cached_attention(q, cache, 0, plan), want)
    # A row's bits do not go by the rows beside it.
    q2 = q.clone()
    q2[2:] *= 3
    assert torch.equal(cached_attention(q2, cache, 0, plan)[:2], want[:2])


def test_agrees_with_packed_attention_over_what_is_read():
    from hyperflow_h3_flash_amd import AttentionPlan, packed_attention
    cache, plan, q, *_ , got = run_attention([2, 130, 1], [700, 300, 64], 8, 4, 128, causal=True)
    k, v = cache_read(cache, 0, plan)
    ref = packed_attention(q, k, v, AttentionPlan([2, 130, 1], [700, 300, 64], heads=8, kv_heads=4, head_dim=128,
                                                  causal=True)).double()
    assert ((got.double() - ref).abs() <= 4 * U.UNIT[BF] * ref.abs() + 0.02).all()


# --------------------------------------------------------------------------------------------- forks, moves and copies

def test_forks_write_apart_and_compaction_moves():
    cache = KVCache(2, 2, 64, 40, page_size=32)
    a = cache.new()
    k, v = keys(1, 100, 2, 64, BF), keys(2, 100, 2, 64, BF)
    first = cache.plan([a], [70])
    for layer in range(2):
        cache_append(cache, layer, k[:70], v[:70], first)
    b, c = cache.fork(a), cache.fork(a)
    with pytest.raises(ValueError, match="forked"):
        cache_append(cache, 0, k[:70], v[:70], first)
    assert torch.equal(cache_read(cache, 0, first)[0].double(), C.held(k[:70]))  # it still reads
    tails = {r: (keys(10 + r, 20, 2, 64, BF), keys(20 + r, 20, 2, 64, BF)) for r in (a, b, c)}
    step = cache.plan([a, b, c], [20, 20, 20])
    assert len({cache.table(r)[2] for r in (a, b, c)}) == 3 and len({cache.table(r)[0] for r in (a, b, c)}) == 1
    for layer in range(2):
        cache_append(cache, layer, torch.cat([tails[r][0] for r in (a, b, c)]), torch.cat([tails[r][1] for r in (a, b, c)]),
                     step)
    x = cache.new()
    cache.plan([x], [320])
    cache.free(a)

    def whole():
        for layer in range(2):
            got = cache_read(cache, layer, cache.plan([b, c], [0, 0]))
            for i, held in enumerate((k, v)):
                want = torch.cat([C.held(torch.cat([held[:70], tails[r][i]])) for r in (b, c)])
                assert torch.equal(got[i].double(), want)

    whole()
    cache.free(x)
    old = cache.plan([b, c], [0, 0])
    used = cache.compact()
    assert used == cache.pages - cache.free_pages and max(p for r in (b, c) for p in cache.table(r)) < used
    with pytest.raises(ValueError, match="moved"):
        cache_read(cache, 0, old)
    whole()
    assert cache.compact() == used


@pytest.mark.parametrize("layers,pages,shape,moves", [(1, 4, (16,), 1), (3, 700, (1040,), 300), (47, 40, (64 * 8 * 136,), 13),
                                                      (2, 9, (3, 16400), 4)])
def test_pages_copied(layers, pages, shape, moves):
    gen = torch.Generator().manual_seed(pages)
    pool = torch.randint(0, 256, (layers, pages, *shape), generator=gen, dtype=torch.uint8).cuda()
    order = torch.randperm(pages, generator=gen).tolist()
    src, dst = order[:moves], order[moves:2 * moves]
    src[0] = src[-1]  # a page may be copied to several
    want = pool.clone()
    want[:, dst] = want[:, src]
    assert copy_pages(pool, src, dst) is pool and torch.equal(pool, want)
    copy_pages(pool, [], [])
    assert torch.equal(pool, want)
    if layers > 1:  # every second layer of a larger pool, of another type
        view = pool.view(torch.int16)[::2]
        want = view.clone()
        want[:, dst] = want[:, src]
        copy_pages(view, src, dst)
        assert torch.equal(view, want)


# ---------------------------------------------------------------------------------------------- streams, graphs, threads

def test_another_stream_and_a_graph():
    cache, requests, k, v = filled([700, 40, 300], 2, 128, spare=1)
    k2, v2 = keys(21, 4, 2, 128, BF), keys(22, 4, 2, 128, BF)
    q = rnd(23, 130, 8, 128).to(BF)
    plan = cache.plan(requests, [1, 2, 127], new_lengths=[1, 2, 1], heads=8, causal=True)

    def step():
        cache_append(cache, 0, k2, v2, plan)
        return cached_attention(q, cache, 0, plan), *cache_read(cache, 0, plan)

    want = [t.clone() for t in step()]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
        copy_pages(cache.data, [cache.table(requests[0])[-1]], [cache.pages - 1])
    for i in range(4):
        q.copy_(rnd(30 + i, 130, 8, 128).to(BF))
        k2.copy_(keys(40 + i, 4, 2, 128, BF))
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in out]
        eager = step()
        assert all(torch.equal(a, b) for a, b in zip(kept, eager)), i
        assert torch.equal(cache.data[0, -1], cache.data[0, cache.table(requests[0])[-1]])


def test_caches_of_inference_mode_and_others():
    for outer, inner in ((torch.inference_mode, torch.no_grad), (torch.no_grad, torch.inference_mode)):
        with outer():
            cache = KVCache(1, 2, 32, 6)
            request = cache.new()
        with inner():
            k, v = keys(1, 100, 2, 32, BF), keys(2, 100, 2, 32, BF)
            plan = cache.plan([request], [100], causal=True)
            cache_append(cache, 0, k, v, plan)
            cache.fork(request)
            cache.plan([request], [1])
            got = cache_read(cache, 0, cache.plan([request], [0]))
            assert torch.equal(got[0][:100].double(), C.held(k))
            ref, bound = C.attention(k, k, v, [100], [100], True, 32 ** -0.5)
            other = KVCache(1, 2, 32, 2)
            step = other.plan([other.new()], [100], causal=True)
            cache_append(other, 0, k, v, step)
            U.check(cached_attention(k, other, 0, step), ref, bound)


def test_two_threads_on_one_stream():
    cache, requests, k, v = filled([9000, 3000], 2, 128)
    plan = cache.plan(requests, [1, 100], new_lengths=[0, 0], heads=8, causal=True)
    assert plan.ws_bytes > 0
    qs = [rnd(i, 101, 8, 128).to(BF) for i in range(2)]
    want = [cached_attention(q, cache, 0, plan) for q in qs]
    torch.cuda.synchronize()
    wrong = []

    def loop(i):
        for _ in range(100):
            if not torch.equal(cached_attention(qs[i], cache, 0, copy.copy(plan)), want[i]):
                wrong.append(i)

    threads = [threading.Thread(target=loop, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong

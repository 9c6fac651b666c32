"""The attention block's operators on the gfx950 kernels against plain 64-bit forms (block_utils.py), at the sizes, masks
and layouts where they can go wrong."""

from __future__ import annotations

import pytest
import torch

import block_utils as U
from hyperflow_h3_flash_amd import AdapterPlan, AttentionPlan, RotaryAxes, adapter_add, packed_attention, qk_norm_rope

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _name(request):
    print(f"case {request.node.name}", flush=True)


def rnd(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).cuda()


# ------------------------------------------------------------------------------------------------- norms and rotation

@pytest.mark.parametrize("T", [1, 2, 7, 64, 257])
@pytest.mark.parametrize("hq,hk,D,dims,interleaved,norm,dtype", [
    (4, 2, 128, (44, 42, 42), True, True, BF),
    (3, 1, 128, (128,), False, False, HF),
    (5, 5, 64, (16, 24, 24), False, True, HF),
    (2, 1, 96, (32, 32), True, True, BF),      # channels after the rotated ones, lanes of a head idle
    (1, 1, 80, (16,), False, True, BF),
    (2, 2, 16, (16,), True, True, BF),
    (7, 3, 256, (64, 96, 96), False, True, BF),
    (33, 9, 128, (64,), False, False, BF),
])
def test_norm_and_rotation(T, hq, hk, D, dims, interleaved, norm, dtype):
    wide = (3 * rnd(T, T, (hq + 2 * hk) * D)).to(dtype)
    q, k = wide[:, :hq * D].view(T, hq, D), wide[:, hq * D:(hq + hk) * D].view(T, hk, D)
    positions = torch.randint(0, 5000, (T, len(dims)), generator=torch.Generator().manual_seed(7)).int().cuda()
    w = (1 + 0.3 * rnd(5, 2, D)).to(dtype) if norm else (None, None)
    rotary = RotaryAxes(dims, theta=1e4, interleaved=interleaved)
    got = qk_norm_rope(q, k, positions, rotary, q_weight=w[0], k_weight=w[1], norm=norm)
    for g, x, wt, name in zip(got, (q, k), w, "qk"):
        U.check(g, *U.rotate(x, wt, positions, dims, 1e4, interleaved, norm), name)


@pytest.mark.parametrize("kind", ["int32", "int64", "float32"])
def test_positions_of_every_type_and_size(kind):
    T, dims = 40, (32, 32, 64)
    positions = torch.randint(-3000000, 3000000, (T, 3), generator=torch.Generator().manual_seed(1))
    positions = (positions / 8 if kind == "float32" else positions).to(getattr(torch, kind)).cuda()
    q = rnd(2, T, 3, 128).to(BF)
    got, none = qk_norm_rope(q, None, positions, RotaryAxes(dims, theta=500.0), norm=False)
    assert none is None
    U.check(got, *U.rotate(q, None, positions, dims, 500.0, True, False))


def test_norm_alone_and_float32_weights_and_zero_rows():
    q = rnd(3, 50, 4, 64).to(HF)
    q[5] = 0
    w = 1 + rnd(4, 64)
    got, _ = qk_norm_rope(q, None, None, None, q_weight=w, eps=1e-5)
    U.check(got, *U.rotate(q, w, None, None, 1.0, True, True, 1e-5))
    assert (got[5] == 0).all()


def test_in_place_strided_outputs_and_unaligned_inputs():
    T, hq, hk, D, dims = 33, 4, 2, 64, (32, 32)
    rotary = RotaryAxes(dims, interleaved=False)
    base = rnd(6, T * (hq + 2 * hk) * D + 8).to(BF)
    positions = torch.arange(2 * T).view(T, 2).cuda()
    for shift in (0, 1, 3):
        wide = base[shift:shift + T * (hq + 2 * hk) * D].clone() if shift == 0 else \
            base.clone()[shift:shift + T * (hq + 2 * hk) * D]
        wide = wide.view(T, (hq + 2 * hk), D)
        q, k, v = wide[:, :hq], wide[:, hq:hq + hk], wide[:, hq + hk:].clone()
        want = [U.rotate(x, None, positions, dims, 1e4, False, True) for x in (q, k)]
        out = qk_norm_rope(q, k, positions, rotary, out=(q, k))
        assert out[0] is q and out[1] is k
        for g, w in zip(out, want):
            U.check(g, *w)
        assert torch.equal(wide[:, hq + hk:], v)  # what lies between stays


def test_heads_first_layout():
    q = rnd(8, 6, 70, 128).to(BF).transpose(0, 1)  # [T, H, D] of a [H, T, D] tensor
    positions = torch.arange(70).cuda()
    got, _ = qk_norm_rope(q, None, positions, RotaryAxes((128,)))
    U.check(got, *U.rotate(q, None, positions[:, None], (128,), 1e4, True, True))


def test_rotation_of_no_tokens():
    got = qk_norm_rope(rnd(1, 0, 4, 64).to(BF), rnd(1, 0, 2, 64).to(BF), torch.zeros(0, 1).int().cuda(), RotaryAxes((64,)))
    assert got[0].shape == (0, 4, 64) and got[1].shape == (0, 2, 64)


# ---------------------------------------------------------------------------------------------------------- attention

def attend(seed, q_lens, kv_lens, hq, hk, D, causal, dtype, scale=None, spread=1.5):
    q = (spread * rnd(seed, sum(q_lens), hq, D)).to(dtype)
    k = (spread * rnd(seed + 1, sum(kv_lens), hk, D)).to(dtype)
    v = (rnd(seed + 2, sum(kv_lens), hk, D) + 0.5).to(dtype)
    plan = AttentionPlan(q_lens, kv_lens, heads=hq, kv_heads=hk, head_dim=D, causal=causal)
    got = packed_attention(q, k, v, plan, scale=scale)
    U.check(got, *U.attention(q, k, v, q_lens, kv_lens, causal, D ** -0.5 if scale is None else scale))
    return q, k, v, plan, got


LENGTHS = [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 321]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("n", LENGTHS)
def test_lengths_around_the_tiles(n, causal):
    attend(n, [n], [n], 2, 1, 128, causal, BF)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("D", [16, 32, 48, 64, 80, 96, 112, 128])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_head_widths_and_types(D, dtype, causal):
    attend(D, [70, 1, 150], [70, 1, 150], 3, 3, D, causal, dtype)


@pytest.mark.parametrize("hq,hk", [(1, 1), (5, 1), (8, 2), (7, 7), (12, 4), (40, 1), (16, 1)])
def test_head_groups(hq, hk):
    attend(hq, [50, 3, 129], [50, 3, 129], hq, hk, 64, True, BF)


def test_packed_ragged_with_empty_sequences():
    attend(1, [0, 5, 64, 0, 200, 1], [7, 5, 64, 0, 200, 0], 4, 2, 64, False, BF)
    attend(2, [3, 0, 64, 17], [0, 0, 10, 40], 4, 4, 128, True, HF)  # queries without a key; more queries than keys


@pytest.mark.parametrize("causal", [False, True])
def test_no_keys_at_all_and_no_queries_at_all(causal):
    out = attend(3, [3, 200], [0, 0], 4, 2, 128, causal, BF)[4]
    assert not out.any()
    assert attend(4, [0, 0], [5, 70], 4, 2, 64, causal, HF)[4].shape == (0, 4, 64)
    assert attend(5, [], [], 4, 2, 64, causal, HF)[4].shape == (0, 4, 64)


@pytest.mark.parametrize("hq,hk", [(8, 8), (32, 8), (16, 1), (12, 12)])
def test_single_tokens_against_caches(hq, hk):
    kv = [1, 2, 63, 64, 65, 1000, 4097, 300]
    attend(hq, [1] * 8, kv, hq, hk, 128, True, BF)


@pytest.mark.parametrize("q,kv", [(1, 20000), (5, 9000), (130, 6000), (33, 2049)])
def test_few_rows_over_many_keys_are_cut_and_joined(q, kv):
    _, _, _, plan, _ = attend(q, [q], [kv], 4, 2, 128, True, BF)
    assert plan.ws_bytes > 0


def test_cross_attention_and_scale():
    attend(4, [300, 77], [20, 513], 3, 3, 96, False, BF, scale=0.3)


def test_sharp_scores_and_rising_maxima():
    """Scores far beyond the range of the weights, rising along the keys so that the running maximum is passed in every
    tile, and falling."""
    n, D = 700, 64
    ramp = torch.linspace(0, 60, n).cuda()
    for order in (ramp, ramp.flip(0)):
        q = torch.zeros(n, 1, D, device="cuda").to(BF)
        q[..., 0] = 8.0
        k = rnd(3, n, 1, D).to(BF)
        k[:, 0, 0] = order.to(BF)
        v = rnd(4, n, 1, D).to(BF)
        plan = AttentionPlan([n], heads=1, head_dim=D, causal=True)
        U.check(packed_attention(q, k, v, plan), *U.attention(q, k, v, [n], [n], True, D ** -0.5))


def test_lowest_values_and_infinities_of_unseen_keys():
    """Keys and values behind a query, and of other sequences, may hold anything."""
    lens, H, D = [100, 30, 200], 2, 64
    q, k, v = (rnd(i, sum(lens), H, D).to(BF) for i in range(3))
    plan = AttentionPlan(lens, heads=H, head_dim=D, causal=True)
    clean = packed_attention(q, k, v, plan)
    for bad in (float("inf"), float("-inf"), float("nan"), torch.finfo(BF).min, torch.finfo(BF).max):
        for where in (90, 129, 250):
            for t in (k, v):
                kept = t[where].clone()
                t[where, 1, ::3] = bad
                got = packed_attention(q, k, v, plan)
                rows = torch.ones(sum(lens), dtype=torch.bool)
                first, end = (0, 100) if where < 100 else (100, 130) if where < 130 else (130, 330)
                rows[where:end] = False
                assert torch.equal(got[rows], clean[rows]), (bad, where)
                assert torch.equal(got[:, 0], clean[:, 0])
                t[where] = kept
    assert torch.equal(packed_attention(q, k, v, plan), clean)


def test_values_that_are_seen_show():
    lens, D = [90], 64
    q, k, v = (rnd(i, 90, 1, D).to(BF) for i in range(3))
    v[70, 0, 3], v[71, 0, 3], v[72, 0, 5] = float("inf"), float("-inf"), float("nan")
    got = packed_attention(q, k, v, AttentionPlan(lens, heads=1, head_dim=D, causal=True))
    assert got[:70].isfinite().all()
    assert (got[70, 0, 3] == float("inf")) and got[71:, 0, 3].isnan().all()
    assert got[:72, 0, 5].isfinite().all() and got[72:, 0, 5].isnan().all()
    rest = [i for i in range(D) if i not in (3, 5)]
    assert got[:, 0, rest].isfinite().all()


def test_unseen_values_in_cut_rows():
    q, k, v = rnd(1, 40, 4, 64).to(BF), rnd(2, 5000, 2, 64).to(BF), rnd(3, 5000, 2, 64).to(BF)
    plan = AttentionPlan([40], [5000], heads=4, kv_heads=2, head_dim=64, causal=True)
    clean = packed_attention(q, k, v, plan)
    v[4980:] = float("nan")
    assert torch.equal(packed_attention(q, k, v, plan)[:20], clean[:20])


def test_strides_of_caches_and_projections():
    lens, H, D = [40, 90], 4, 64
    n = sum(lens)
    wide = rnd(1, n, 3 * H, D).to(BF)
    views = [wide[:, i * H:(i + 1) * H] for i in range(3)]
    plan = AttentionPlan(lens, heads=H, head_dim=D)
    ref = U.attention(*views, lens, lens, False, D ** -0.5)
    U.check(packed_attention(*views, plan), *ref)
    heads_first = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in views]
    out = torch.empty(n, 2 * H, D, device="cuda", dtype=BF)
    got = packed_attention(*heads_first, plan, out=out[:, ::2])
    assert got.data_ptr() == out.data_ptr()
    U.check(got, *ref)
    odd = [torch.empty(t.numel() + 1, device="cuda", dtype=BF)[1:].view(t.shape).copy_(t) for t in views]
    U.check(packed_attention(*odd, plan), *ref)
    shared = views[1][:, :1].expand(n, H, D)  # one key head seen as all
    U.check(packed_attention(views[0], shared, shared, plan), *U.attention(views[0], shared, shared, lens, lens, False,
                                                                           D ** -0.5))


def test_offsets_past_32_bits():
    """A cache of which one sequence begins past 2^32 bytes, with strides of a wide row."""
    rows, D = 70000, 64
    cache = torch.zeros(rows, 34816, device="cuda", dtype=BF)  # 4.9 GB
    k, v = cache[:, 512:512 + D].unsqueeze(1), cache[:, 34816 - D:].unsqueeze(1)
    k.copy_(rnd(1, rows, 1, D).to(BF))
    v.copy_(rnd(2, rows, 1, D).to(BF))
    lens = [65000, 5000]
    q = rnd(3, 5, 2, D).to(BF)
    plan = AttentionPlan([2, 3], lens, heads=2, kv_heads=1, head_dim=D, causal=True)
    U.check(packed_attention(q, k, v, plan), *U.attention(q, k, v, [2, 3], lens, True, D ** -0.5))


def test_same_bits_every_time():
    *_, plan, first = attend(9, [1, 40, 1], [9000, 3000, 5], 8, 2, 128, True, BF)
    q, k, v = (1.5 * rnd(9, 42, 8, 128)).to(BF), (1.5 * rnd(10, 12005, 2, 128)).to(BF), (rnd(11, 12005, 2, 128) + 0.5).to(BF)
    for _ in range(3):
        assert torch.equal(packed_attention(q, k, v, plan), first)


# ----------------------------------------------------------------------------------------------------------- adapters

def adapt(seed, ids, lens, adapters, r, K, N, dtype, scaled=True, spread=1.0):
    M = sum(lens)
    x, y = (spread * rnd(seed, M, K)).to(dtype), rnd(seed + 1, M, N).to(dtype)
    down, up = (rnd(seed + 2, adapters, r, K) / K ** 0.5).to(dtype), (rnd(seed + 3, adapters, N, r) / r ** 0.5).to(dtype)
    scale = 0.5 + rnd(seed + 4, adapters).abs() if scaled else None
    plan = AdapterPlan(ids, lens, adapters=adapters)
    ref = U.adapters(y, x, down, up, ids, lens, scale)
    kept = y.clone()
    got = adapter_add(y, x, down, up, plan, scale=scale)
    U.check(got, *ref)
    assert torch.equal(y, kept)
    again = adapter_add(y, x, down, up, plan, scale=scale, out=y)
    assert again is y and torch.equal(y, got)
    none = torch.tensor([a for a, n in zip(ids, lens) for _ in range(n)]) < 0
    assert torch.equal(got[none], kept[none])


@pytest.mark.parametrize("M", [1, 2, 31, 32, 33, 63, 64, 65, 130, 700])
def test_rows_around_the_tiles(M):
    adapt(M, [0], [M], 1, 16, 256, 192, BF)


@pytest.mark.parametrize("r", [8, 16, 24, 32, 40, 64, 96, 128, 136, 256, 512])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_ranks(r, dtype):
    adapt(r, [1, 0, -1, 1], [40, 33, 5, 1], 2, r, 320, 136, dtype)


@pytest.mark.parametrize("K,N", [(8, 8), (64, 64), (72, 1), (1000, 72), (5120, 64), (4104, 999), (264, 3), (128, 65), (56, 7168)])
def test_widths(K, N):
    adapt(K + N, [0, 2, -1], [70, 3, 9], 3, 32, K, N, BF)


@pytest.mark.parametrize("r", [16, 64, 128, 200])
def test_few_rows_over_a_deep_k(r):
    adapt(r, [0, 1], [9, 40], 2, r, 14344, 72, BF)


@pytest.mark.parametrize("r", [8, 64, 96, 160])
def test_many_rows(r):
    adapt(r, [1, 0, -1, 1], [17000, 15990, 33, 40], 2, r, 200, 136, BF)


def test_many_requests_in_any_order():
    ids = [(i * 7) % 12 - 1 for i in range(150)]
    adapt(5, ids, [1 + i % 3 for i in range(150)], 11, 16, 512, 256, BF, scaled=False)
    adapt(6, [-1, -1], [5, 60], 2, 16, 512, 256, BF)  # none has one
    adapt(7, [1, 0, 1], [0, 0, 5], 2, 16, 512, 256, HF)  # requests of no rows


def test_large_and_small_intermediates():
    for spread in (1e-3, 300.0):  # the intermediate's fp16 range is not the result's
        adapt(8, [0, 1], [20, 50], 2, 24, 640, 200, HF, spread=spread)
    adapt(9, [0], [40], 1, 24, 640, 200, BF, spread=1e10)


def test_rows_with_infinities_stay_alone():
    M, K, N, r = 40, 256, 128, 16
    x, y = rnd(1, M, K).to(BF), rnd(2, M, N).to(BF)
    down, up = rnd(3, 1, r, K).to(BF), rnd(4, 1, N, r).to(BF)
    plan = AdapterPlan([0], [M], adapters=1)
    clean = adapter_add(y, x, down, up, plan)
    x[7, 3], x[9, 0] = float("inf"), float("nan")
    got = adapter_add(y, x, down, up, plan)
    rows = [i for i in range(M) if i not in (7, 9)]
    assert torch.equal(got[rows], clean[rows])
    assert not got[7].isfinite().any() and got[9].isnan().all()


def test_adapter_strides():
    M, K, N, r = 50, 256, 136, 16
    wide_x, wide_y = rnd(1, M, K + 8).to(BF), rnd(2, M, N + 5).to(BF)
    down, up = rnd(3, 2, r, K).to(BF), rnd(4, 2, N, r).to(BF)
    ids, lens = [1, -1, 0], [20, 10, 20]
    plan = AdapterPlan(ids, lens, adapters=2)
    for x, y in ((wide_x[:, 8:], wide_y[:, :N]), (wide_x[:, 1:K + 1], wide_y[:, 5:]),
                 (wide_x[:, :K].t().contiguous().t(), wide_y[:, :N].t().contiguous().t())):
        ref = U.adapters(y, x, down, up, ids, lens, None)
        U.check(adapter_add(y, x, down, up, plan), *ref)
        out = torch.zeros(M, N + 3, device="cuda", dtype=BF)
        adapter_add(y, x, down, up, plan, out=out[:, 3:])
        U.check(out[:, 3:], *ref)
        assert (out[:, :3] == 0).all()


# -------------------------------------------------------------------------------------------------------------- module

def test_block_equals_its_parts():
    from test_block import make_block

    block = make_block(dim=512, heads=8, kv_heads=2, head_dim=64, group=256, device="cuda")
    lengths, ids = [5, 300, 1, 64], [1, -1, 0, 1]
    T = sum(lengths)
    x = rnd(1, T, 512).to(BF)
    positions = torch.randint(0, 50, (T, 2), generator=torch.Generator().manual_seed(3)).cuda()
    rotary = RotaryAxes((32, 32))
    plan = AttentionPlan(lengths, heads=8, kv_heads=2, head_dim=64)
    adapters = AdapterPlan(ids, lengths, adapters=2)
    got = block(x, plan, positions=positions, rotary=rotary, adapters=adapters)
    qkv = block.qkv_adapters(block.qkv(x), x, adapters).view(T, 12, 64)
    q, k = qk_norm_rope(qkv[:, :8], qkv[:, 8:10], positions, rotary, q_weight=block.norm_q, k_weight=block.norm_k)
    o = packed_attention(q, k, qkv[:, 10:], plan)
    U.check(o, *U.attention(q, k, qkv[:, 10:], lengths, lengths, False, 64 ** -0.5))
    o = o.view(T, 512)
    assert torch.equal(block.out_adapters(block.out(o), o, adapters), got)


# ------------------------------------------------------------------------------------------------------------ streams

def test_plans_on_another_stream_and_in_a_graph():
    lens = [1, 30, 1]
    kv = [3000, 30, 700]
    q, k, v = rnd(1, 32, 8, 64).to(BF), rnd(2, sum(kv), 2, 64).to(BF), rnd(3, sum(kv), 2, 64).to(BF)
    positions = torch.arange(32).cuda()
    rotary = RotaryAxes((64,), device="cuda")
    plan = AttentionPlan(lens, kv, heads=8, kv_heads=2, head_dim=64, causal=True)
    down, up = rnd(4, 2, 16, 512).to(BF), rnd(5, 2, 512, 16).to(BF)
    adapters = AdapterPlan([1, -1, 0], lens, adapters=2)

    def step():
        turned, _ = qk_norm_rope(q, None, positions, rotary)
        o = packed_attention(turned, k, v, plan).view(32, 512)
        return adapter_add(o, o, down, up, adapters)

    want = step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for i in range(4):
        q.copy_(rnd(10 + i, 32, 8, 64).to(BF))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, step()), i

"""The attention block's operators as programs call them: from several threads, with copied plans, in place between other
layers, beyond 2^31 elements."""

from __future__ import annotations

import copy
import math
import pickle
import threading

import pytest
import torch

import block_utils as U
from hyperflow_h3_flash_amd import (AdapterPlan, AttentionPlan, Int8RotLinear, RotaryAxes, adapter_add,
                                    packed_attention, qk_norm_rope)

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _name(request):
    print(f"case {request.node.name}", flush=True)


def rnd(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).cuda()


def test_two_threads_on_one_stream():
    """Each thread's cut attention and joined adapters use workspaces of their own, though both launch on one stream."""
    kv = [9000, 3000]
    plan = AttentionPlan([1, 9], kv, heads=8, kv_heads=2, head_dim=128, causal=True)
    adapters = AdapterPlan([0, -1, 1], [9, 2, 21], adapters=2)
    assert plan.ws_bytes > 0
    down, up = (rnd(1, 2, 160, 14336) / 120).to(HF), (rnd(2, 2, 72, 160) / 12).to(HF)
    work = []
    for i in range(2):
        q, k, v = rnd(3 + i, 10, 8, 128).to(BF), rnd(5 + i, sum(kv), 2, 128).to(BF), rnd(7 + i, sum(kv), 2, 128).to(BF)
        x, y = rnd(9 + i, 32, 14336).to(HF), rnd(11 + i, 32, 72).to(HF)
        work.append(lambda a=(q, k, v, plan), b=(y, x, down, up, adapters): (packed_attention(*a), adapter_add(*b)))
    want = [w() for w in work]
    torch.cuda.synchronize()
    wrong = []

    def loop(i):
        for _ in range(150):
            if not all(torch.equal(a, b) for a, b in zip(work[i](), want[i])):
                wrong.append(i)

    threads = [threading.Thread(target=loop, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


# ------------------------------------------------------------------------------------------------- results in place

def int8_layer(k, n, seed):
    layer = Int8RotLinear(k, n, 256)
    gen = torch.Generator().manual_seed(seed)
    layer.qweight.copy_(torch.randint(-127, 128, layer.qweight.shape, generator=gen, dtype=torch.int8))
    layer.wscale.fill_(k ** -0.5 / 73)
    return layer.cuda()


@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
@pytest.mark.parametrize("op", ["rotation", "attention", "adapters"])
def test_a_layer_after_an_update_in_place_takes_the_new_values(op, mode):
    """The first of two layers that share one input leaves its codes; the input is updated in place between them."""
    first, second = int8_layer(256, 128, 1), int8_layer(256, 96, 2)
    first.keep_input = True
    try:
        with mode():
            x = rnd(3, 20, 256).to(BF)
            heads = x.view(20, 4, 64)
            first(x)
            assert torch.equal(second(x), second(x.clone()))  # shared, and right while x stays
            first(x)
            if op == "rotation":
                qk_norm_rope(heads, None, torch.arange(20).cuda(), RotaryAxes((64,)), out=(heads, None))
            elif op == "attention":
                packed_attention(heads, heads.clone(), heads.clone(), AttentionPlan([20], heads=4, head_dim=64), out=heads)
            else:
                adapter_add(x, x.clone(), rnd(4, 1, 8, 256).to(BF), rnd(5, 1, 256, 8).to(BF),
                            AdapterPlan([0], [20], adapters=1), out=x)
            assert torch.equal(second(x), second(x.clone()))
    finally:
        Int8RotLinear._last_input.clear()


def test_a_saved_tensor_that_is_overwritten_shows_in_backward():
    y, x = rnd(1, 20, 64).to(BF), rnd(2, 20, 64).to(BF)
    w = torch.ones(64, device="cuda", dtype=BF, requires_grad=True)
    product = y * w  # y is kept for the gradient of w
    adapter_add(y, x, rnd(3, 1, 8, 64).to(BF), rnd(4, 1, 64, 8).to(BF), AdapterPlan([0], [20], adapters=1), out=y)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.sum().backward()


# -------------------------------------------------------------------------------------------------- copies of plans

@pytest.mark.parametrize("copied", [copy.copy, copy.deepcopy, lambda x: pickle.loads(pickle.dumps(x))],
                         ids=["copy", "deepcopy", "pickle"])
def test_copies_outlive_the_plans_and_tables_they_were_made_of(copied):
    kv = [3000, 40]
    held = {"rotary": RotaryAxes((32, 32), device="cuda"),
            "plan": AttentionPlan([2, 3], kv, heads=4, kv_heads=2, head_dim=64, causal=True),
            "adapters": AdapterPlan([1, -1], [2, 3], adapters=2)}
    q, k, v = rnd(1, 5, 4, 64).to(BF), rnd(2, sum(kv), 2, 64).to(BF), rnd(3, sum(kv), 2, 64).to(BF)
    x, down, up = rnd(4, 5, 256).to(BF), rnd(5, 2, 16, 256).to(BF), rnd(6, 2, 256, 16).to(BF)
    positions = torch.arange(10).view(5, 2).cuda()

    def step():
        turned, _ = qk_norm_rope(q, None, positions, held["rotary"])
        o = packed_attention(turned, k, v, held["plan"])
        return adapter_add(o.view(5, 256), x, down, up, held["adapters"])

    want = step()
    for name in list(held):
        held[name] = copied(held[name])
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    taken = [torch.full((1 << 16,), 255, dtype=torch.uint8, device="cuda") for _ in range(20)]  # what was given back
    assert torch.equal(step(), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert torch.equal(got, want) and len(taken) == 20


def test_results_over_the_inputs_are_those_of_a_separate_result():
    """A result may name memory that the call reads: keys, values, the other side's heads, rows of y further on."""
    lens, H, D = [500, 40], 4, 64
    n = sum(lens)
    plan, positions, rotary = AttentionPlan(lens, heads=H, head_dim=D), torch.arange(n).cuda(), RotaryAxes((D,))

    def fresh():
        return [rnd(i, n, H, D).to(BF) for i in range(3)]

    q, k, v = fresh()
    want, (q_want, k_want) = packed_attention(q, k, v, plan), qk_norm_rope(q, k, positions, rotary)
    for name in range(3):
        t = fresh()
        assert torch.equal(packed_attention(*t, plan, out=t[name]), want)
        x = fresh()[0]
        assert torch.equal(packed_attention(x, x, x, plan, out=x), packed_attention(*[fresh()[0]] * 3, plan))
    for out in ((1, 0), (1, 2), (2, 0), (0, 1)):
        t = fresh()
        qk_norm_rope(t[0], t[1], positions, rotary, out=(t[out[0]], t[out[1]]))
        assert torch.equal(t[out[0]], q_want) and torch.equal(t[out[1]], k_want)
    adapters, down, up = AdapterPlan([0, -1], lens, adapters=1), rnd(5, 1, 8, 64).to(BF), rnd(6, 1, 64, 8).to(BF)
    x, rows = rnd(7, n, 64).to(BF), rnd(8, n + 3, 64).to(BF)
    want = adapter_add(rows[:n].clone(), x, down, up, adapters)
    assert torch.equal(adapter_add(rows[:n], x, down, up, adapters, out=rows[3:]), want)
    y = rnd(8, n + 3, 64).to(BF)[:n]
    assert torch.equal(adapter_add(y, x, down, up, adapters, out=x), want)


# ------------------------------------------------------------------------------------------------ attention's weights

@pytest.mark.parametrize("exponent", [14.0, 20.0, 25.0625, 29.0])
@pytest.mark.parametrize("dtype", [HF, BF])
def test_small_weights_beside_a_dominant_one(dtype, exponent):
    """One key that takes nearly all of the weight and 40000 of equal small weights, in tiles of rows that are not cut (a
    share without the dominant key has a maximum of its own). Rounding errs by at most u of a weight where fp16 is normal,
    and by 2^-31 of the largest weight below that: fp16's least step of 2^-24, halved, with weights taken up to 2^6."""
    n, D, M = 40001, 64, 65536
    q = torch.zeros(M, 1, D, device="cuda", dtype=dtype)
    q[..., 0] = 1
    k = torch.zeros(n, 1, D, device="cuda", dtype=dtype)
    k[5, 0, 0] = exponent
    for v in (torch.ones(n, 1, D, device="cuda"), 0.5 + rnd(1, n, 1, D)):
        v = v.to(dtype)
        v[5] = 0
        plan = AttentionPlan([M], [n], heads=1, head_dim=D)
        assert plan.ws_bytes == 0
        scale = math.log(2.0)
        got = packed_attention(q, k, v, plan, scale=scale)
        assert (got == got[0]).all()
        w = torch.exp2(k[:, 0, 0].double() * (scale * math.log2(math.e)))
        w /= w.sum()
        want, size = w @ v[:, 0].double(), w @ v[:, 0].double().abs()
        u = U.UNIT[dtype]
        # A score errs by a few float32 roundings of its size, which moves a weight in proportion; sums run over n keys.
        off = (exponent * (D + 8) + n) * 2.0 ** -24
        lost = 2.0 ** -31 * v[:, 0].double().abs().sum(0) if dtype is HF else 0.0
        U.check(got[0, 0], want, u * want.abs() + (u + off) * size + lost + U.TINY[dtype], str(exponent))


def test_scores_of_no_weight_in_fp16():
    """The smallest scales make every weight one; one of them is a share's, joined."""
    for rows, n in ((300, 70), (3, 5000)):
        q, k, v = rnd(1, rows, 1, 64).to(HF), rnd(2, n, 1, 64).to(HF), rnd(3, n, 1, 64).to(HF)
        plan = AttentionPlan([rows], [n], heads=1, head_dim=64)
        for scale in (1e-6, 1e-30, 1e-37):
            U.check(packed_attention(q, k, v, plan, scale=scale), *U.attention(q, k, v, [rows], [n], False, scale))


@pytest.mark.parametrize("top", [60.0, 3000.0])
@pytest.mark.parametrize("rows,n,heads", [(700, 700, 200), (700, 700, 1), (3, 6000, 1), (40, 3000, 1)])
@pytest.mark.parametrize("dtype", [HF, BF])
def test_rising_and_falling_scores(dtype, rows, n, heads, top):
    """The maximum moves in every tile, or stays that of the first, in whole tiles of rows and in shares of cut ones."""
    D = 64
    plan = AttentionPlan([rows], [n], heads=heads, head_dim=D, causal=True)
    assert (plan.ws_bytes > 0) == (heads == 1)
    ramp = torch.linspace(0, top, n).cuda()
    q = torch.zeros(rows, 1, D, device="cuda", dtype=dtype)
    q[..., 0] = 8.0  # scores are the ramp at the scale of 1 / 8
    for order in (ramp, ramp.flip(0), -ramp, ramp[torch.arange(n).cuda() * 7919 % n]):
        k, v = rnd(3, n, 1, D).to(dtype), rnd(4, n, 1, D).to(dtype)
        k[:, 0, 0] = order.to(dtype)
        got = packed_attention(*(t.expand(-1, heads, D) for t in (q, k, v)), plan)
        assert (got == got[:, :1]).all()
        U.check(got[:, :1], *U.attention(q, k, v, [rows], [n], True, D ** -0.5))


@pytest.mark.parametrize("rows,n", [(90, 90), (3, 6000)])
def test_infinities_and_nan_in_fp16(rows, n):
    """Values that are seen show, in whole and in cut rows; those that are not leave no trace."""
    D = 64
    q, k, v = rnd(1, rows, 1, D).to(HF), rnd(2, n, 1, D).to(HF), rnd(3, n, 1, D).to(HF)
    plan = AttentionPlan([rows], [n], heads=1, head_dim=D, causal=True)
    clean = packed_attention(q, k, v, plan)
    last = rows - 2  # the last query but one sees all keys but the last
    v[n - 1, 0, 3], v[n - 2, 0, 4], v[0, 0, 5] = float("inf"), float("-inf"), float("nan")
    got = packed_attention(q, k, v, plan)
    assert got[rows - 1, 0, 3] == float("inf") and torch.equal(got[:last + 1, 0, 3], clean[:last + 1, 0, 3])
    assert (got[last:, 0, 4] == float("-inf")).all() and torch.equal(got[:last, 0, 4], clean[:last, 0, 4])
    assert got[:, 0, 5].isnan().all() and torch.equal(got[:, 0, 6:], clean[:, 0, 6:])


# ------------------------------------------------------------------------------------------------- past 2^31 elements

def test_adapters_past_32_bits():
    M, K, N, r = 150016, 14400, 15368, 16
    gen = torch.Generator(device="cuda").manual_seed(1)
    x, y = (torch.randn(M, n, generator=gen, device="cuda", dtype=BF) for n in (K, N))
    assert x.numel() > 2 ** 31 and y.numel() > 2 ** 31
    down, up = (rnd(2, 2, r, K) / K ** 0.5).to(BF), (rnd(3, 2, N, r) / r ** 0.5).to(BF)
    lens, ids = [70000, 16, M - 70016], [0, -1, 1]
    plan = AdapterPlan(ids, lens, adapters=2)
    picked = torch.cat([torch.arange(a, a + 40) for a in (0, 69980, 2 ** 31 // N - 20, 2 ** 31 // K - 20, M - 40)]).cuda()
    which = torch.repeat_interleave(torch.tensor(ids), torch.tensor(lens))[picked.cpu()].tolist()
    want = U.adapters(y[picked], x[picked], down, up, which, [1] * len(which), None)
    U.check(adapter_add(y, x, down, up, plan, out=y)[picked], *want)


def test_rotation_past_32_bits():
    T, H, D = 140003, 120, 128
    q = torch.randn(T, H, D, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda", dtype=BF)
    assert q.numel() > 2 ** 31
    positions = torch.arange(T).cuda()
    picked = torch.cat([torch.arange(a, a + 8) for a in (0, 2 ** 31 // (H * D) - 4, T - 8)]).cuda()
    want = U.rotate(q[picked], None, positions[picked, None], (D,), 1e4, True, True)
    U.check(qk_norm_rope(q, None, positions, RotaryAxes((D,)), out=(q, None))[0][picked], *want)


@pytest.mark.parametrize("theta", [1e4, 5.0])
def test_positions_to_the_ends_of_int32(theta):
    positions = torch.tensor([[2 ** 31 - 1], [-2 ** 31], [2 ** 31 - 3], [123456789]]).cuda()
    q = rnd(2, 4, 3, 128).to(HF)
    for p in (positions, positions.int()):
        got, _ = qk_norm_rope(q, None, p, RotaryAxes((128,), theta=theta), norm=False)
        U.check(got, *U.rotate(q, None, positions, (128,), theta, True, False))

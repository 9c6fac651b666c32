"""The norms before and after a block with its gate and residual, on the GPU, against 64 bits."""

from __future__ import annotations

import pytest
import torch

import block_utils as U
import cache_utils as C
from hyperflow_h3_flash_amd import RowPlan, residual_norm

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _name(request):
    print(f"case {request.node.name}", flush=True)


def rnd(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).cuda()


def run(lens, width, norm="rms", post=None, dtype=BF, stream=None, y=True, weights=False, modulated=True, residual=1.0,
        vectors=None, eps=1e-6, mean=0.0, seed=0):
    T, stream, vectors = sum(lens), stream or dtype, vectors or dtype
    x = (2 * rnd(seed + 1, T, width) + mean).to(stream)
    b = (rnd(seed + 2, T, width) + mean).to(dtype) if y else None
    m = (0.5 * rnd(seed + 3, len(lens), 3, width)).to(vectors) if modulated else None
    gate, shift, scale = (None if m is None else m[:, i] for i in range(3))
    w = (1 + 0.2 * rnd(seed + 4, width)).to(vectors) if weights else None
    pw = (1 + 0.2 * rnd(seed + 5, width)).to(vectors) if weights and post else None
    gate = gate if y else None
    rows = RowPlan(lens) if modulated else None
    got = residual_norm(x, b, rows=rows, residual=residual, gate=gate, post_norm=post, post_weight=pw, norm=norm, weight=w,
                        scale=scale, shift=shift, eps=eps, dtype=None if y else dtype)
    groups = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens)).cuda()
    r, n = C.residual_norm(x, b, groups, residual, gate, post, pw, norm, w, scale, shift, eps, dtype)
    if y:
        assert got[0].dtype is stream
        U.check(got[0], *r, f"r of {lens} x {width}")
    else:
        assert got[0] is x
    assert got[1].dtype is dtype
    U.check(got[1], *n, f"n of {lens} x {width}")
    return got


@pytest.mark.parametrize("width", [8, 64, 504, 512, 520, 1024, 1032, 2048, 2056, 4096, 4104, 5376, 6152, 8192, 8200, 12288,
                                   12296, 16384])
@pytest.mark.parametrize("norm,post", [("rms", None), ("layer", "rms")])
def test_widths(width, norm, post):
    run([3, 0, 2], width, norm, post, weights=True, seed=width)


@pytest.mark.parametrize("width", [512, 1024, 2048, 4096, 6144, 8192, 12288, 16384])
@pytest.mark.parametrize("norm,post", [("layer", "rms"), ("rms", "layer")])
@pytest.mark.parametrize("stream,vectors", [(BF, BF), (F32, F32)])
def test_sums_by_the_kernels_own_chains(width, norm, post, stream, vectors, monkeypatch):
    """The widest row of each shape, held to the additions that its sums make one behind the other: 8 terms for each of a lane's
    chunks (1 or 2; 3 with 4 or 8 waves), 6 exchanges, and the row's 1 to 16 waves: at most 16 + 6 + 16 or 24 + 6 + 8. With the
    quotient by the width 39 roundings."""
    monkeypatch.setattr(C, "SUM", 39 * 2.0 ** -24)
    for mean in (0.0, 20.0):
        run([3, 2], width, norm, post, BF, stream, weights=True, vectors=vectors, mean=mean, seed=width)


@pytest.mark.parametrize("norm", ["rms", "layer", None])
@pytest.mark.parametrize("post", ["rms", "layer", None])
@pytest.mark.parametrize("dtype,stream", [(BF, BF), (HF, HF), (BF, F32), (HF, F32)])
def test_kinds_and_types(norm, post, dtype, stream):
    for width in (264, 2560):
        run([1, 4, 6], width, norm, post, dtype, stream, weights=True, residual=0.5)
        run([11], width, norm, post, dtype, stream, modulated=norm is None, vectors=F32)


@pytest.mark.parametrize("T", [1, 2, 3, 4, 5, 63, 1000])
def test_rows(T):
    run([T], 512, "layer")
    run([T], 1544, "rms", y=False)


def test_first_norm_of_a_model():
    run([5, 7], 640, "layer", y=False)
    run([5, 7], 640, "rms", y=False, stream=F32, weights=True)
    run([5, 7], 640, None, y=False, dtype=HF)


def test_last_block_without_a_norm():
    x, y, gate = rnd(1, 9, 640).to(BF), rnd(2, 9, 640).to(BF), rnd(3, 640).to(BF)
    r, n = residual_norm(x, y, gate=gate, norm=None)
    assert n is None
    (want, bound), _ = C.residual_norm(x, y, None, 1.0, gate, None, None, None, None, None, None, 1e-6, BF)
    U.check(r, want, bound)


@pytest.mark.parametrize("norm", ["rms", "layer"])
def test_rows_far_from_zero_and_rows_of_one_value(norm):
    run([6], 5376, norm, mean=300.0, stream=F32)
    x = torch.full((4, 768), 3.0, device="cuda", dtype=BF)
    x[1] = 0.0
    r, n = residual_norm(x, torch.zeros_like(x), norm=norm, eps=1e-6)
    assert torch.equal(r, x)
    want = torch.zeros(4, 768, device="cuda", dtype=torch.float64)
    if norm == "rms":
        want[[0, 2, 3]] = 3.0 / (9.0 + 1e-6) ** 0.5
    U.check(n, want, want.abs() * 2.0 ** -8 + 1e-30)


def test_rows_with_infinities_and_nan_stay_alone():
    x, y = rnd(1, 12, 1024).to(BF), rnd(2, 12, 1024).to(BF)
    clean = residual_norm(x, y, norm="layer")
    x[3, 5], y[7, 1000], x[9, 0] = float("inf"), float("nan"), float("-inf")
    got = residual_norm(x, y, norm="layer")
    rest = [i for i in range(12) if i not in (3, 7, 9)]
    for a, b in zip(got, clean):
        assert torch.equal(a[rest], b[rest])
    assert got[0][3, 5] == float("inf") and got[0][7, 1000].isnan() and got[1][7].isnan().all() and got[1][3].isnan().all()


def test_a_vector_for_all_rows_or_one_a_row():
    x, y = rnd(1, 20, 320).to(BF), rnd(2, 20, 320).to(BF)
    one, many = rnd(3, 320).to(BF), rnd(4, 20, 320).to(BF)
    rows = torch.arange(20, device="cuda")
    r, n = residual_norm(x, y, gate=many, scale=one, shift=many)
    wr, wn = C.residual_norm(x, y, rows, 1.0, many, None, None, "rms", None, one, many, 1e-6, BF)
    U.check(r, *wr)
    U.check(n, *wn)
    a = residual_norm(x, y, rows=RowPlan([20]), gate=one[None], scale=one, shift=one)
    b = residual_norm(x, y, gate=one, scale=one[None], shift=one.expand(20, 320))
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    x1 = x[:1]
    assert torch.equal(residual_norm(x1, y[:1], gate=many[:1])[0], residual_norm(x1, y[:1], gate=many[0])[0])


def test_outputs_in_place_and_strides():
    x, y = rnd(1, 70, 640).to(BF), rnd(2, 70, 640).to(BF)
    want = residual_norm(x, y, norm="layer", residual=0.5)

    def same(got):
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])

    a, b = x.clone(), y.clone()
    v = a._version
    got = residual_norm(a, b, norm="layer", residual=0.5, out=(a, b))
    assert got[0] is a and got[1] is b and a._version > v
    same(got)
    a, b = x.clone(), y.clone()
    same(residual_norm(a, b, norm="layer", residual=0.5, out=(b, a)))
    wide = torch.zeros(70, 4, 640, device="cuda", dtype=BF)
    wide[:, 1], wide[:, 2] = x, y
    same(residual_norm(wide[:, 1], wide[:, 2], norm="layer", residual=0.5, out=(wide[:, 0], wide[:, 3])))
    same(residual_norm(wide[:, 1], wide[:, 2], norm="layer", residual=0.5, out=(wide[:, 2], wide[:, 1])))
    shifted = torch.zeros(71, 640, device="cuda", dtype=BF)
    shifted[:70] = x
    same(residual_norm(shifted[:70], y, norm="layer", residual=0.5, out=(shifted[1:], torch.empty_like(y))))
    odd = torch.zeros(70, 641, device="cuda", dtype=BF)
    odd[:, 1:] = x
    same(residual_norm(odd[:, 1:], y, norm="layer", residual=0.5))
    xs = x[:1].expand(70, 640)
    r, _ = residual_norm(xs, y)
    assert torch.equal(r, residual_norm(xs.contiguous(), y)[0])
    single = residual_norm(odd[:1, 1:], y[:1], norm="layer", residual=0.5)  # one row, at any stride and start
    assert torch.equal(single[0], want[0][:1]) and torch.equal(single[1], want[1][:1])
    single = residual_norm(odd[:1].new_zeros(1, 649)[:, :640], y[:1, :640])
    assert torch.equal(single[0], y[:1])
    one = torch.empty_like(x)
    with pytest.raises(ValueError, match="places of their own"):
        residual_norm(x, y, norm="layer", residual=0.5, out=(one, one.view(70, 640)))
    with pytest.raises(ValueError, match="places of their own"):
        residual_norm(x[:69], y[:69], norm="layer", out=(one[:69], one[1:]))


def test_a_tensor_past_2_31_elements():
    T, width = 140000, 16384
    x = torch.zeros(T, width, device="cuda", dtype=BF)
    x[-1], x[0] = rnd(1, width).to(BF), rnd(2, width).to(BF)
    y = rnd(3, 1, width).to(BF).expand(T, width)
    r, n = residual_norm(x, y, norm="rms")
    for i in (0, -1, 131072):
        a, b = residual_norm(x[i][None], y[:1].contiguous(), norm="rms")
        assert torch.equal(r[i], a[0]) and torch.equal(n[i], b[0])


def test_more_rows_than_one_launch_takes():
    T = (1 << 25) + 70001
    x = torch.zeros(T, 8, device="cuda", dtype=BF)
    x[-1], x[1 << 25], x[(1 << 25) - 1] = 3.0, 5.0, 7.0
    gate = torch.ones(T, 8, device="cuda", dtype=BF)
    gate[-1] = 2.0
    r, n = residual_norm(x, x, gate=gate)
    assert r[-1].eq(9).all() and r[1 << 25].eq(10).all() and r[(1 << 25) - 1].eq(14).all() and n[-1].eq(1).all()
    assert r.count_nonzero() == 24 and n.count_nonzero() == 24


def test_no_rows():
    e = torch.empty(0, 64, device="cuda", dtype=BF)
    r, n = residual_norm(e, e.clone(), rows=RowPlan([0, 0]), gate=torch.zeros(2, 64, device="cuda", dtype=BF))
    assert r.shape == n.shape == (0, 64)


def test_another_stream_and_a_graph():
    lens = [40, 3]
    rows = RowPlan(lens)
    x, y = rnd(1, 43, 1280).to(BF), rnd(2, 43, 1280).to(BF)
    m = rnd(3, 2, 3, 1280).to(BF)

    def step():
        return residual_norm(x, y, rows=rows, gate=m[:, 0], scale=m[:, 1], shift=m[:, 2], norm="layer")

    want = step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(3):
        x.copy_(rnd(10 + i, 43, 1280).to(BF))
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(kept, step()))

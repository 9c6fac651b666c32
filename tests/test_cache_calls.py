"""What the 4-bit cache's operators and the residual norms do around their launches, without a GPU: host tensors that say they
lie on a device, and a library that looks at a launch's parameters instead of launching."""

from __future__ import annotations

import contextlib
import sys
import weakref

import pytest
import torch

import hyperflow_h3_flash_amd as hf
from hyperflow_h3_flash_amd import KVCache, RowPlan, _native, block, kv_cache
from test_block_calls import on_device

BF = torch.bfloat16
norms = sys.modules["hyperflow_h3_flash_amd.residual_norm"]
PACKERS = {"hf_cache_append": _native.CACHE_APPEND_ARGS, "hf_cache_read": _native.CACHE_READ_ARGS,
           "hf_cached_attention": _native.CACHED_ATTENTION_ARGS, "hf_copy_pages": _native.COPY_PAGES_ARGS,
           "hf_residual_norm": _native.RESIDUAL_NORM_ARGS}


class Launches:
    def __init__(self):
        self.lib, self.seen, self.look = _native.block_library(), [], lambda name, args: None

    def __getattr__(self, name):
        if name not in PACKERS:
            return getattr(self.lib, name)

        def launch(packed):
            args = PACKERS[name].unpack(packed)
            self.seen.append((name, args))
            self.look(name, args)
            return _native.HF_OK

        return launch


@pytest.fixture
def launches(monkeypatch):
    stub = Launches()
    for module in (block, kv_cache, norms):
        for name, what in (("_lib", lambda device: stub), ("_raw_stream", lambda index: 0),
                           ("_on", lambda device: contextlib.nullcontext()),
                           ("_current", lambda index, device: contextlib.nullcontext())):
            if hasattr(module, name):
                monkeypatch.setattr(module, name, what)
    return stub


def rnd(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def cache_and_plan(q_lengths, kv_lengths, heads=4):
    cache = KVCache(2, 2, 32, 400, device="cpu")
    cache._index = 0
    requests = [cache.new() for _ in kv_lengths]
    cache.plan(requests, kv_lengths)
    plan = cache.plan(requests, q_lengths, new_lengths=[0] * len(q_lengths), heads=heads, causal=True)
    plan._lay_out(_native.block_library(), 256)
    return cache, plan


def test_the_workspace_lives_until_its_kernels_are_launched(launches, monkeypatch):
    cache, plan = cache_and_plan([1, 9], [9000, 300])
    made, empty = [], torch.empty

    def tracked(*args, **kwargs):
        t = empty(*args, **kwargs)
        made.append((t.data_ptr(), t.numel() * t.element_size(), weakref.ref(t)))
        return t

    def look(name, args):
        ws, nbytes = args[11], args[12]
        assert nbytes == plan.ws_bytes > 0 and any(p == ws and n == nbytes and r() is not None for p, n, r in made)

    launches.look = look
    monkeypatch.setattr(torch, "empty", tracked)
    hf.cached_attention(on_device(rnd(1, 10, 4, 32).to(BF)), cache, 1, plan)
    assert [name for name, _ in launches.seen] == ["hf_cached_attention"]
    assert launches.seen[0][1][3] == cache.data[1].data_ptr()


def test_attention_writes_in_place_and_never_over_other_queries(launches):
    cache, plan = cache_and_plan([1, 9], [900, 300])
    wide = on_device(torch.zeros(10, 9, 32, dtype=BF))
    q = wide[:, 1:5]
    for out, direct in ((q, True), (wide[:, 5:9], True), (wide[:, 2:6], False), (wide[:, 0:4], False)):
        hf.cached_attention(q, cache, 0, plan, out=out)
        args = launches.seen[-1][1]
        assert (args[4] == out.data_ptr()) == direct and args[0] == q.data_ptr() and args[1:3] == (288, 32)
        if direct:
            assert args[5:7] == (288, 32)
        else:
            assert not wide.data_ptr() <= args[4] < wide.data_ptr() + wide.numel() * 2


def test_appended_tensors_that_vectors_cannot_read_are_copied(launches):
    cache, plan = cache_and_plan([1], [5])
    step = cache.plan([0], [3])
    step._lay_out(_native.block_library(), 256)
    odd = on_device(torch.zeros(3, 2, 33, dtype=BF))[..., 1:]
    fused = on_device(torch.zeros(3, 8, 32, dtype=BF))
    version = cache.data._version
    hf.cache_append(cache, 1, odd, fused[:, 6:], step)
    k, kt, kh, v, vt, vh, pages, *_ = launches.seen[-1][1]
    assert k % 16 == 0 and k != odd.data_ptr() and (kt, kh) == (64, 32)
    assert (v, vt, vh) == (fused[:, 6:].data_ptr(), 256, 32) and pages == cache.data[1].data_ptr()
    assert cache.data._version > version


def test_residual_norms_write_where_nothing_else_is_read(launches):
    T, width = 20, 64
    wide = on_device(torch.zeros(T, 6, width, dtype=BF))
    x, y = wide[:, 1], wide[:, 2]
    shifted = on_device(torch.zeros(T + 1, width, dtype=BF))
    for given, outs, direct in (
            ((x, y), (x, y), (True, True)), ((x, y), (y, x), (True, True)), ((x, y), (wide[:, 0], wide[:, 5]), (True, True)),
            ((shifted[:T], y), (shifted[1:], wide[:, 5]), (False, True)), ((x, shifted[1:]), (x, shifted[:T]), (True, False))):
        hf.residual_norm(*given, out=outs)
        args = launches.seen[-1][1]
        assert (args[0], args[2]) == tuple(t.data_ptr() for t in given)
        assert tuple(args[i] == o.data_ptr() for i, o in zip((4, 6), outs)) == direct
    vector = wide[0, 3]  # a vector that a result would overwrite
    hf.residual_norm(x, y, shift=vector, out=(wide[:, 3], wide[:, 4]))
    assert launches.seen[-1][1][4] != wide[:, 3].data_ptr() and launches.seen[-1][1][6] == wide[:, 4].data_ptr()


def test_modulation_strides(launches):
    T, width = 5, 64
    x, y = on_device(rnd(1, T, width).to(BF)), on_device(rnd(2, T, width).to(BF))
    m = on_device(rnd(3, 2, 6, width).to(BF))
    rows = RowPlan([2, 3], device="cpu")
    rows._index, rows.data = 0, block._Resident(rows.groups, torch.device("cpu"))
    hf.residual_norm(x, y, rows=rows, gate=m[:, 2], scale=m[:, 1], shift=m[0, 0])
    args = launches.seen[-1][1]
    assert args[8:14] == (m[:, 2].data_ptr(), 6 * width, m[:, 1].data_ptr(), 6 * width, m[0, 0].data_ptr(), 0)
    assert args[16] == rows.groups.data_ptr() and args[17:20] == (2, T, width) and args[22] == 0
    hf.residual_norm(x, y, gate=m[:1, 2].expand(T, width))
    args = launches.seen[-1][1]
    assert args[8:10] == (m[0, 2].data_ptr(), 0) and args[16] == 0 and args[17] == T and args[22] == 1 and args[24] == 0
    hf.residual_norm(x, y, gate=m[:1, 2], scale=m[1, 1].float())  # all vectors in float32
    args = launches.seen[-1][1]
    assert args[8] != m[0, 2].data_ptr() and args[9] == args[11] == 0 and args[24] == 1


def test_page_numbers_do_not_wrap(launches):
    pool = on_device(torch.zeros(2, 8, 16, dtype=torch.uint8))
    for src, dst in (([1 << 32], [1]), ([1], [(1 << 32) + 2]), ([-1], [1])):
        with pytest.raises(ValueError, match="pages must be"):
            hf.copy_pages(pool, src, dst)
    assert not launches.seen
    hf.copy_pages(pool, [1, 1], [2, 3])
    assert launches.seen[-1][1][1:5] == (2, 128, 8, 16)

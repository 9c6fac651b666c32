"""What the attention block's operators do around their launches, without a GPU: host tensors that say they lie on a
device, and a library that looks at a launch's parameters instead of launching."""

from __future__ import annotations

import contextlib
import copy
import ctypes
import heapq
import io
import os
import pickle
import random
import re
import struct
import weakref

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

from hyperflow_h3_flash_amd import (AdapterPlan, AttentionBlock, AttentionPlan, Int8RotLinear, RotaryAxes, adapter_add,
                                    packed_attention, qk_norm_rope)
from hyperflow_h3_flash_amd import _native, block

BF = torch.bfloat16


class OnDevice(torch.Tensor):
    """A host tensor that says it lies on device 0."""

    is_cuda = property(lambda self: True)

    def get_device(self):
        return 0


def on_device(t):
    return t.as_subclass(OnDevice)


def rnd(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


class Launches:
    """The library with its launches replaced: each appends (name, parameters) and runs ``look`` on the parameters."""

    def __init__(self):
        self.lib = _native.block_library()
        self.seen = []
        self.look = lambda name, args: None

    def __getattr__(self, name):
        packers = {"hf_qk_norm_rope_call": _native.ROPE_ARGS, "hf_attention_call": _native.ATTENTION_ARGS,
                   "hf_adapter_add_call": _native.ADAPTER_ARGS}
        if name not in packers:
            return getattr(self.lib, name)

        def launch(packed):
            args = packers[name].unpack(packed)
            self.seen.append((name, args))
            self.look(name, args)
            return _native.HF_OK

        return launch


@pytest.fixture
def launches(monkeypatch):
    if not os.path.exists(_native.BLOCK_LIB_PATH):
        pytest.fail(f"{_native.BLOCK_LIB_PATH} not built: run __graft_entry__.build()")
    stub = Launches()
    monkeypatch.setattr(block, "_lib", lambda device: stub)
    monkeypatch.setattr(block, "_raw_stream", lambda index: 0)
    monkeypatch.setattr(block, "_on", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(block, "_current", lambda index, device: contextlib.nullcontext())
    return stub


def attention_plan(q_lens, kv_lens, heads, kv_heads, head_dim, causal=False):
    plan = AttentionPlan(q_lens, kv_lens, heads=heads, kv_heads=kv_heads, head_dim=head_dim, causal=causal, device="cpu")
    lib = _native.block_library()
    q, kv = block._array(ctypes.c_int64, plan.q_lengths), block._array(ctypes.c_int64, plan.kv_lengths)
    plan._fill("hf_attention_plan", lib, plan.device, ctypes.addressof(q), ctypes.addressof(kv), len(q_lens), heads,
               kv_heads, head_dim, causal, 256)
    plan.ws_bytes = lib.hf_attention_ws_bytes(plan.data.host_address, plan.bytes)
    plan._index = 0
    return plan


def adapter_plan(ids, lengths, adapters):
    plan = AdapterPlan(ids, lengths, adapters=adapters, device="cpu")
    lib = _native.block_library()
    ids_c, lens_c = block._array(ctypes.c_int32, plan.ids), block._array(ctypes.c_int64, plan.lengths)
    plan._fill("hf_adapter_plan", lib, plan.device, ctypes.addressof(ids_c), ctypes.addressof(lens_c), len(ids), adapters,
               256)
    plan._index = 0
    return plan


# ---------------------------------------------------------------------------------------------------------- workspaces

WS = {"hf_attention_call": (16, 17), "hf_adapter_add_call": (15, 16)}  # places of the workspace and its bytes


@pytest.mark.parametrize("call", ["attention", "adapters"])
def test_the_workspace_lives_until_its_kernels_are_launched(launches, monkeypatch, call):
    """A block given back before the launch could be handed to another thread's call on the same stream."""
    made = []
    empty = torch.empty

    def tracked(*args, **kwargs):
        t = empty(*args, **kwargs)
        made.append((t.data_ptr(), t.numel() * t.element_size(), weakref.ref(t)))
        return t

    def look(name, args):
        ws, nbytes = (args[i] for i in WS[name])
        assert nbytes > 0 and any(p == ws and n >= nbytes and alive() is not None for p, n, alive in made)

    launches.look = look
    if call == "attention":
        plan = attention_plan([1], [9000], 4, 2, 64)
        q, k, v = (on_device(rnd(i, n, h, 64).to(BF)) for i, (n, h) in enumerate(((1, 4), (9000, 2), (9000, 2))))
        monkeypatch.setattr(torch, "empty", tracked)
        packed_attention(q, k, v, plan)
    else:
        plan = adapter_plan([0, -1], [9, 2], 1)
        x, y = on_device(rnd(1, 11, 64).to(BF)), on_device(rnd(2, 11, 48).to(BF))
        down, up = on_device(rnd(3, 1, 8, 64).to(BF)), on_device(rnd(4, 1, 48, 8).to(BF))
        monkeypatch.setattr(torch, "empty", tracked)
        adapter_add(y, x, down, up, plan)
    assert len(launches.seen) == 1


# ------------------------------------------------------------------------------------------------- results in place

def in_place_calls():
    """(what is written, call) of each operator writing into tensors that were there."""
    qkv = on_device(rnd(1, 6, 4, 64).to(BF))
    q, k, v = qkv[:, :2], qkv[:, 2:3], qkv[:, 3:]
    plan = attention_plan([6], [6], 2, 1, 64)
    adapters = adapter_plan([0, -1], [4, 2], 1)
    x, y, wide = (on_device(rnd(i, 6, n).to(BF)) for i, n in ((2, 64), (3, 48), (4, 56)))
    down, up = on_device(rnd(5, 1, 8, 64).to(BF)), on_device(rnd(6, 1, 48, 8).to(BF))
    return {
        "rotation": ((q, k), lambda: qk_norm_rope(q, k, None, None, out=(q, k))),
        "rotation of queries alone": ((q,), lambda: qk_norm_rope(q, None, None, None, out=(q, None))),
        "attention": ((q,), lambda: packed_attention(q, k, v, plan, out=q)),
        "adapters": ((y,), lambda: adapter_add(y, x, down, up, adapters, out=y)),
        "adapters into a slice": ((wide,), lambda: adapter_add(y, x, down, up, adapters, out=wide[:, :48])),
    }


@pytest.mark.parametrize("name", ["rotation", "rotation of queries alone", "attention", "adapters",
                                  "adapters into a slice"])
def test_results_in_place_move_the_version(launches, name):
    """Autograd's check of saved tensors and the codes that INT8 layers share go by a tensor's version."""
    written, call = in_place_calls()[name]
    before = [t._version for t in written]
    call()
    assert launches.seen and all(t._version > n for t, n in zip(written, before))


@pytest.mark.parametrize("name", ["rotation", "attention", "adapters", "adapters into a slice"])
def test_results_in_place_drop_codes_of_inference_tensors(launches, name):
    """Inference tensors have no version, so codes that a layer left of one go when it is written; others stay."""
    cache = Int8RotLinear._last_input
    try:
        with torch.inference_mode():
            written, call = in_place_calls()[name]
            assert written[0].is_inference()
            for x, stays in ((written[0], False), (rnd(9, 4, 4), True)):
                cache.clear()
                cache.update(x=x, version=None, value=None)
                call()
                assert bool(cache) is stays
    finally:
        cache.clear()


def test_new_results_leave_the_inputs_versions(launches):
    q, k = on_device(rnd(1, 6, 2, 64).to(BF)), on_device(rnd(2, 6, 1, 64).to(BF))
    before = q._version, k._version
    qk_norm_rope(q, k, None, None)
    packed_attention(q, k, k, attention_plan([6], [6], 2, 1, 64))
    assert launches.seen and (q._version, k._version) == before


# -------------------------------------------------------------------------------------------------- copies of plans

def by_pickle(x):
    return pickle.loads(pickle.dumps(x))


def by_torch_save(x):
    held = io.BytesIO()
    torch.save(x, held)
    held.seek(0)
    return torch.load(held, weights_only=False)


@pytest.mark.parametrize("copied", [copy.copy, copy.deepcopy, by_pickle, by_torch_save])
def test_copies_of_plans_and_tables_point_at_memory_of_their_own(launches, copied):
    """Every address that a call with a copy passes on lies in a tensor that the copy itself keeps."""
    rotary = RotaryAxes((32, 32))
    rotary.tables(torch.device("cpu"))
    attention, adapters = attention_plan([3], [700], 2, 1, 64), adapter_plan([0], [3], 1)
    rotary2, attention2, adapters2 = (copied(x) for x in (rotary, attention, adapters))
    keep = [r.device_copy.clone() for r in rotary.tables(torch.device("cpu"))]
    q, k = on_device(rnd(1, 3, 2, 64).to(BF)), on_device(rnd(2, 700, 1, 64).to(BF))
    rotary2._tables[0] = rotary2.tables(torch.device("cpu"))
    qk_norm_rope(q, None, torch.zeros(3, 2, dtype=torch.int32).as_subclass(OnDevice), rotary2)
    packed_attention(q, k, k, attention2)
    x, y = on_device(rnd(3, 3, 64).to(BF)), on_device(rnd(4, 3, 48).to(BF))
    adapter_add(y, x, on_device(rnd(5, 1, 8, 64).to(BF)), on_device(rnd(6, 1, 48, 8).to(BF)), adapters2)
    (_, rope), (_, attend), (_, adapt) = launches.seen
    tables = rotary2.tables(torch.device("cpu"))
    assert list(rope[18:20]) == [t.device_copy.data_ptr() for t in tables]
    assert all(torch.equal(t.device_copy, want) for t, want in zip(tables, keep))
    for seen, at, plan, first in ((attend, 13, attention2, attention), (adapt, 12, adapters2, adapters)):
        assert list(seen[at:at + 2]) == [plan.data.host.data_ptr(), plan.data.device_copy.data_ptr()]
        assert torch.equal(plan.data.host, first.data.host)


def test_a_copied_module_keeps_its_rotation(launches):
    module = torch.nn.Linear(2, 2)
    module.rotary = RotaryAxes((64,))
    module.rotary.tables(torch.device("cpu"))
    other = copy.deepcopy(module)
    want = [t.device_copy.clone() for t in module.rotary.tables(torch.device("cpu"))]
    del module
    for t, w in zip(other.rotary.tables(torch.device("cpu")), want):
        assert t.on(0) == t.device_copy.data_ptr() and torch.equal(t.device_copy, w)


def test_a_plan_made_elsewhere_is_uploaded_at_its_first_use(launches):
    """A pickled plan may be loaded where its device is not: it waits for a call."""
    plan = by_pickle(attention_plan([3], [700], 2, 1, 64))
    assert plan.data.device_copy is None
    assert plan.data.on(0) == plan.data.device_copy.data_ptr()


# --------------------------------------------------------------------------------------------- results over the inputs

def test_attention_never_writes_where_it_still_reads(launches):
    """Workgroups read keys and values long after others have written rows of the result."""
    qkv = on_device(rnd(1, 6, 4, 64).to(BF))
    q, k, v = qkv[:, :2], qkv[:, 2:3], qkv[:, 3:]
    plan, alike = attention_plan([6], [6], 2, 1, 64), attention_plan([6], [6], 2, 2, 64)
    whole = on_device(rnd(2, 6, 2, 64).to(BF))
    halves = on_device(rnd(3, 6, 2, 3, 64).to(BF))  # q, k and v of a head side by side
    heads_first = on_device(rnd(4, 4, 6, 64).to(BF)).transpose(0, 1)
    shifted = on_device(rnd(5, 8, 2, 64).to(BF))
    for args, out, direct in (
        ((q, k, v, plan), q, True), ((q, k, v, plan), on_device(rnd(6, 6, 2, 64).to(BF)), True),
        ((*halves.unbind(2), alike), halves[:, :, 0], True),
        ((heads_first[:, :2], heads_first[:, 2:3], heads_first[:, 3:], plan), heads_first[:, :2], True),
        ((whole, whole, whole, alike), whole, False), ((q, whole, qkv[:, 2:], alike), whole, False),
        ((q, qkv[:, 2:], whole, alike), whole, False), ((q, k, v, plan), qkv[:, 1:3], False),
        ((shifted[:6], whole, whole, alike), shifted[2:], False),  # the queries of another row
        ((*halves.unbind(2), alike), halves[:, :, 1], False),
    ):
        packed_attention(*args, out=out)
        assert (launches.seen[-1][1][9] == out.data_ptr()) is direct


def test_rotation_and_adapters_never_write_where_they_still_read(launches):
    q, k, other = (on_device(rnd(i, 6, 2, 64).to(BF)) for i in range(3))
    long = on_device(rnd(3, 9, 2, 64).to(BF))
    for args, out, direct in (
        ((q, k), (q, k), (True, True)), ((q, k), (q, other), (True, True)), ((q, k), (q.view(6, 2, 64), k), (True, True)),
        ((q, k), (k, q), (False, False)), ((q, k), (k, other), (False, True)), ((q, k), (other, q), (True, False)),
        ((long[:6], None), (long[1:7], None), (False, True)),
    ):
        qk_norm_rope(*args, None, None, out=out)
        seen = launches.seen[-1][1]
        assert (seen[8] == out[0].data_ptr()) is direct[0]
        assert out[1] is None or (seen[11] == out[1].data_ptr()) is direct[1]
    plan = adapter_plan([0, -1], [4, 2], 1)
    x, wide, rows = on_device(rnd(4, 6, 64).to(BF)), on_device(rnd(5, 6, 128).to(BF)), on_device(rnd(6, 9, 64).to(BF))
    down, up = on_device(rnd(7, 1, 8, 64).to(BF)), on_device(rnd(8, 1, 64, 8).to(BF))
    y = wide[:, :64]
    for y, out, direct in ((y, y, True), (y, wide[:, :64], True), (y, wide[:, 64:], True), (y, wide[:, 8:72], False),
                           (rows[:6], rows[3:], False), (y, x, True)):  # x is read before anything is written
        adapter_add(y, x, down, up, plan, out=out)
        assert (launches.seen[-1][1][8] == out.data_ptr()) is direct


def test_places_that_are_called_apart_share_no_element():
    rng = random.Random(3)

    def elements(place):
        address, rows, heads, row, head, width = place
        return [address // 2 + i * row + j * head + k for i in range(rows) for j in range(heads) for k in range(width)]

    def place():
        head, heads = rng.choice([0, 8, 16, 24, 32, 48]), rng.randint(0, 3)
        row = rng.choice([0, 8, 16, 48, 64, 96, head * max(heads, 1), head * 3])
        return 16 * rng.randint(0, 30), rng.randint(0, 4), heads, row, head, rng.choice([8, 16])

    told = 0
    for _ in range(20000):
        a, b = place(), place()
        if rng.random() < 0.6:
            b = (*b[:3], *a[3:])
        mine, others = elements(a), elements(b)
        if block._apart(a, b):
            told += 1
            assert not set(mine) & set(others), (a, b)
        if block._spread(a):
            assert len(set(mine)) == len(mine), a
    assert told > 10000


def test_results_that_overlap_themselves_are_refused(launches):
    """As torch's own operations refuse to write several values to one place."""
    q = on_device(rnd(1, 6, 2, 64).to(BF))
    out = on_device(torch.zeros(1, 2, 64, dtype=BF)).expand(6, 2, 64)
    for bad in (lambda: qk_norm_rope(q, None, None, None, out=(out, None)),
                lambda: packed_attention(q, q, q, attention_plan([6], [6], 2, 2, 64), out=out),
                lambda: adapter_add(q[:, 0], q[:, 1], on_device(rnd(3, 1, 8, 64).to(BF)), on_device(rnd(4, 1, 64, 8).to(BF)),
                                    adapter_plan([0], [6], 1), out=out[:, 0])):
        with pytest.raises(RuntimeError, match="single memory location|overlap"):
            bad()


# ----------------------------------------------------------------------------------------------------- forward only

def operators(device):
    """Each operator as (name, its tensors by name, call)."""
    move = on_device if device else (lambda t: t)
    t = {n: move(rnd(i, *shape).to(BF)) for i, (n, shape) in enumerate(
        (("q", (6, 2, 64)), ("k", (6, 1, 64)), ("v", (6, 1, 64)), ("w", (64,)), ("x", (6, 32)), ("y", (6, 48)),
         ("down", (1, 8, 32)), ("up", (1, 48, 8)), ("out", (6, 2, 64)), ("out2", (6, 48))))}
    t["positions"], t["scale"] = move(torch.arange(6.0)), move(torch.ones(1))
    plan, adapters = attention_plan([6], [6], 2, 1, 64), adapter_plan([0], [6], 1)
    if not device:
        plan._index = adapters._index = -1
    rotary = RotaryAxes((64,))
    rotary._tables[0] = rotary.tables(torch.device("cpu"))
    return (
        (("q", "k", "positions", "w", "out"), t, lambda t: qk_norm_rope(
            t["q"], t["k"], t["positions"], rotary, q_weight=t["w"], out=(t["out"], t["k"]))),
        (("q", "k", "v", "out"), t, lambda t: packed_attention(t["q"], t["k"], t["v"], plan, out=t["out"])),
        (("x", "y", "down", "up", "scale", "out2"), t, lambda t: adapter_add(
            t["y"], t["x"], t["down"], t["up"], adapters, scale=t["scale"], out=t["out2"])),
    )


@pytest.mark.parametrize("device", [False, True], ids=["host", "device"])
def test_what_would_have_to_be_differentiated_is_refused(launches, device):
    """Gradients and forward-mode tangents of every tensor that a call takes, its result's among them."""
    for names, tensors, call in operators(device):
        call(tensors)
        for name in names:
            leaf = tensors[name].clone().requires_grad_()
            with pytest.raises(RuntimeError, match="forward only"):
                call({**tensors, name: leaf})
            with torch.no_grad():
                call({**tensors, name: leaf})
            with forward_ad.dual_level():
                dual = forward_ad.make_dual(tensors[name].clone(), torch.ones_like(tensors[name]))
                with pytest.raises(RuntimeError, match="forward only"):
                    call({**tensors, name: dual})
                with pytest.raises(RuntimeError, match="forward only"), torch.no_grad():  # which keeps tangents
                    call({**tensors, name: dual})
                call(tensors)


def test_the_block_refuses_what_would_have_to_be_differentiated():
    from test_block import make_block

    block = make_block()
    plan = AttentionPlan([4], heads=4, kv_heads=2, head_dim=16, device="cpu")
    x = rnd(1, 4, 64).to(BF)
    want = block(x, plan)
    assert not want.requires_grad
    with torch.no_grad():
        assert torch.equal(block(x.clone().requires_grad_(), plan), want)
    with pytest.raises(RuntimeError, match="forward only"):
        block(x.clone().requires_grad_(), plan)
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward only"):
        block(forward_ad.make_dual(x, torch.ones_like(x)), plan)
    block.norm_q.requires_grad_()
    with pytest.raises(RuntimeError, match="forward only"):
        block(x, plan)


# ----------------------------------------------------------------------------------------------------------- the block

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32, torch.float64])
def test_adapters_of_a_converted_module(dtype):
    """`nn.Module.to` converts every floating point parameter; the INT8 layers of the block take theirs back too."""
    from test_block import make_block

    block = make_block()
    lengths = [3, 4]
    x = rnd(1, 7, 64).to(BF)
    plan = AttentionPlan(lengths, heads=4, kv_heads=2, head_dim=16, device="cpu")
    adapters = AdapterPlan([1, 0], lengths, adapters=2, device="cpu")
    for bank in (block.qkv_adapters, block.out_adapters):
        bank.scale.copy_(torch.tensor([0.25, 0.75]))  # values that every type holds, as those of the wscale that follows
    for layer in (block.qkv, block.out):
        layer.wscale.fill_(2.0 ** -9)
    block.norm_q.copy_(1 + torch.arange(16) / 32)
    for p in (block.qkv_adapters.down, block.qkv_adapters.up, block.out_adapters.down, block.out_adapters.up):
        p.copy_(p.clamp(-1, 1).mul(64).round().div(64))
    want = block(x, plan, adapters=adapters)
    got = block.to(dtype)(x, plan, adapters=adapters)
    assert got.dtype is BF and torch.equal(got, want)


def block_and_its_projections():
    from test_block import make_block

    block = make_block(adapters=0)
    layers = [Int8RotLinear(64, n, 16) for n in (64, 32, 32)]
    for layer, rows in zip(layers, (slice(0, 64), slice(64, 96), slice(96, 128))):
        layer.qweight.copy_(block.qkv.qweight[rows])
        layer.wscale.copy_(block.qkv.wscale[rows])
    return block, (*layers, block.out, 16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_block_of_a_models_projections_has_its_norms(recwarn, dtype):
    block, projections = block_and_its_projections()
    assert not (block.norm_q == 1).all() and not (block.norm_k == 1).all()
    plan, x = AttentionPlan([5], heads=4, kv_heads=2, head_dim=16, device="cpu"), rnd(1, 5, 64).to(BF)
    weights = {"norm_q": torch.nn.Parameter(block.norm_q.to(dtype)), "norm_k": torch.nn.Parameter(block.norm_k.to(dtype))}
    again = AttentionBlock.from_projections(*projections, **weights)
    assert torch.equal(again(x, plan), block(x, plan))
    assert not any(p.requires_grad or p.is_meta for p in again.parameters()) and weights["norm_q"].requires_grad
    none = AttentionBlock.from_projections(*projections, qk_norm=False)
    assert none.norm_q is None and none.norm_k is None
    ones = AttentionBlock.from_projections(*projections, qk_norm=True)
    assert (ones.norm_q == 1).all() and (ones.norm_k == 1).all()
    assert not [w for w in recwarn.list if w.category is UserWarning]


def test_a_block_of_projections_alone_says_what_it_takes_for_the_norms():
    _, projections = block_and_its_projections()
    with pytest.warns(UserWarning, match="norm_q"):
        block = AttentionBlock.from_projections(*projections)
    assert (block.norm_q == 1).all() and (block.norm_k == 1).all()


def test_refusals_of_norms_that_do_not_fit():
    block, projections = block_and_its_projections()
    w = torch.ones(16)
    for bad in ({"norm_q": w}, {"norm_k": w}, {"norm_q": w, "norm_k": w, "qk_norm": False},
                {"norm_q": torch.ones(64), "norm_k": torch.ones(32)}, {"norm_q": w, "norm_k": torch.ones(1, 16)}):
        with pytest.raises(ValueError):
            AttentionBlock.from_projections(*projections, **bad)


@pytest.mark.parametrize("device", [False, True], ids=["host", "device"])
def test_numbers_outside_of_float32_are_refused_as_arguments(launches, device):
    """scale and eps reach the kernels in float32."""
    move = on_device if device else (lambda t: t)
    q = move(rnd(1, 6, 2, 64).to(BF))
    plan = attention_plan([6], [6], 2, 2, 64)
    if not device:
        plan._index = -1
    for value in (1e39, float("inf")):
        with pytest.raises(ValueError, match="scale"):
            packed_attention(q, q, q, plan, scale=value)
    with pytest.raises(ValueError, match="eps"):
        qk_norm_rope(q, None, None, None, eps=1e39)
    packed_attention(q, q, q, plan, scale=1e38)
    qk_norm_rope(q, None, None, None, eps=1e38)


# --------------------------------------------------------------------------------------------------- built kernels

def kernel_metadata(path):
    """{kernel's symbol: {field: number}} of the code object's notes: MessagePack maps with sorted keys, in which a kernel's
    register counts follow its symbol."""
    data = open(path, "rb").read()
    found = {}
    for m in re.finditer(rb"\.symbol(?:[\xa0-\xbf]|\xd9.)([\x21-\x7e]+?)\.kd", data, flags=re.S):
        fields = {}
        for name in (b".vgpr_count", b".vgpr_spill_count"):
            at = data.index(name, m.end()) + len(name)
            size = {0xcc: 1, 0xcd: 2, 0xce: 4}.get(data[at], 0)
            fields[name.decode()[1:]] = int.from_bytes(data[at + 1:at + 1 + size], "big") if size else data[at]
        found[m.group(1).decode()] = fields
    return found


def test_three_workgroups_of_narrow_heads_share_a_compute_unit():
    """A SIMD's 512 vector registers hold three waves of up to 168: attention on heads of at most 64 depends on it."""
    kernels = {n: f for n, f in kernel_metadata(_native.BLOCK_LIB_PATH).items() if "attention_kernel" in n}
    assert len(kernels) == 6
    for name, fields in kernels.items():
        assert fields["vgpr_spill_count"] == 0 and 0 < fields["vgpr_count"] <= 256, (name, fields)
        if "ELi2E" in name:
            assert fields["vgpr_count"] <= 168, (name, fields)


# ----------------------------------------------------------------------------------------------------- uneven batches

@pytest.mark.parametrize("q,kv,heads,kv_heads", [
    ([1] * 65, [131072] + [1000] * 64, 8, 8), ([1] * 60, [65536] * 4 + [2000] * 56, 32, 8),
    ([1] * 1001, [131072] + [1000] * 1000, 8, 8),
])
def test_a_long_cache_among_many_others_is_cut(q, kv, heads, kv_heads):
    """No single share of a tile's keys takes more than twice an equal share of all the work, and places that take the items
    as they come end within one and a half (a part costs its start and its sums, two tiles of keys)."""
    plan = attention_plan_bytes(q, kv, heads, kv_heads)
    items, joins = struct.unpack_from("2i", plan, 20)
    item = np.frombuffer(plan, np.int32, items * 12, 128).reshape(items, 12)
    tiles = ((item[:, 6] - item[:, 5] + 63) // 64).tolist()
    places = [0] * 512
    for n in tiles:
        heapq.heapreplace(places, places[0] + n + 2)
    share = -(-sum(tiles) // 512)
    assert joins > 0 and max(tiles) <= 2 * share and max(places) <= 1.5 * share
    # every key of every tile of rows once
    rows = {}
    for i in item.tolist():
        rows.setdefault((i[0], i[4], i[7]), []).append((i[5], i[6]))
    for parts in rows.values():
        parts.sort()
        assert parts[0][0] == 0 and all(a[1] == b[0] for a, b in zip(parts, parts[1:]))


def attention_plan_bytes(q, kv, heads, kv_heads):
    lib = _native.block_library()
    qa, ka = (ctypes.c_int64 * len(q))(*q), (ctypes.c_int64 * len(kv))(*kv)
    args = qa, ka, len(q), heads, kv_heads, 128, 1, 256
    held = ctypes.create_string_buffer(lib.hf_attention_plan(*args, None, 0))
    assert lib.hf_attention_plan(*args, held, len(held)) == len(held)
    return held.raw

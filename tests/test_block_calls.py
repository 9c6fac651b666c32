"""What the attention block's operators do around their launches, without a GPU: host tensors that say they lie on a
device, and a library that looks at a launch's parameters instead of launching."""

from __future__ import annotations

import contextlib
import ctypes
import os
import weakref

import pytest
import torch

from hyperflow_h3_flash_amd import AdapterPlan, AttentionPlan, RotaryAxes, adapter_add, packed_attention, qk_norm_rope
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
    plan.ws_bytes = lib.hf_attention_ws_bytes(plan._host, plan.bytes)
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

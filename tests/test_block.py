"""The attention block's operators without a GPU: the host path against the plain 64-bit forms, the refusals, the C ABI's
surface and argument checks, and the planners' layouts."""

from __future__ import annotations

import ctypes
import os
import re
import struct

import numpy as np
import pytest
import torch

import block_utils as U
from hyperflow_h3_flash_amd import AdapterPlan, AttentionPlan, RotaryAxes, adapter_add, packed_attention, qk_norm_rope
from hyperflow_h3_flash_amd import _native

BF, HF = torch.bfloat16, torch.float16
HEADER = os.path.join(_native.REPO_DIR, "include", "hf_block.h")


def rnd(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_native.BLOCK_LIB_PATH):
        pytest.fail(f"{_native.BLOCK_LIB_PATH} not built: run __graft_entry__.build()")
    return _native.block_library()


# ---------------------------------------------------------------------------------------------------------- host path

@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dims,D", [((44, 42, 42), 128), ((16,), 80), ((64,), 64)])
def test_host_norm_and_rotation(dims, D, interleaved):
    q, k = (2 * rnd(1, 9, 3, D)).to(BF), rnd(2, 9, 1, D).to(BF)
    positions = torch.randint(0, 4000, (9, len(dims)), generator=torch.Generator().manual_seed(3))
    w = 1 + 0.2 * rnd(4, D)
    out = (torch.empty_like(q), torch.empty_like(k))
    got = qk_norm_rope(q, k, positions, RotaryAxes(dims, theta=300.0, interleaved=interleaved), q_weight=w.to(BF),
                       k_weight=w, out=out)
    assert got is out
    U.check(got[0], *U.rotate(q, w.to(BF), positions, dims, 300.0, interleaved, True))
    U.check(got[1], *U.rotate(k, w, positions, dims, 300.0, interleaved, True))


def test_a_rotation_turns_by_the_position_difference():
    """Scores of rotated queries and keys depend on the difference of their positions on every axis."""
    rotary = RotaryAxes((16, 24, 24))
    q, k = rnd(1, 1, 1, 64).to(HF), rnd(2, 1, 1, 64).to(HF)

    def score(a, b):
        at = lambda p: torch.tensor([p], dtype=torch.int32)  # noqa: E731
        x, _ = qk_norm_rope(q, None, at(a), rotary, norm=False)
        y, _ = qk_norm_rope(k, None, at(b), rotary, norm=False)
        return float((x.double() * y.double()).sum())

    size = float(q.double().abs().sum() * k.double().abs().max())
    assert abs(score((5, 7, 9), (1, 2, 3)) - score((14, 25, 106), (10, 20, 100))) < 4 * U.UNIT[HF] * size


@pytest.mark.parametrize("causal", [False, True])
def test_host_attention(causal):
    q_lens, kv_lens = [0, 5, 12, 3, 4], [7, 5, 2, 0, 9]
    q, k, v = rnd(1, 24, 4, 32).to(BF), rnd(2, 23, 2, 32).to(BF), rnd(3, 23, 2, 32).to(BF)
    plan = AttentionPlan(q_lens, kv_lens, heads=4, kv_heads=2, head_dim=32, causal=causal, device="cpu")
    out = torch.full_like(q, 9.0)
    got = packed_attention(q, k, v, plan, scale=0.4, out=out)
    assert got is out
    U.check(got, *U.attention(q, k, v, q_lens, kv_lens, causal, 0.4))


def test_host_attention_keeps_unseen_values_out():
    q, k, v = (rnd(i, 10, 1, 16).to(BF) for i in range(3))
    plan = AttentionPlan([10], heads=1, head_dim=16, causal=True, device="cpu")
    clean = packed_attention(q, k, v, plan)
    v[6, 0, 2] = float("inf")
    k[8] = float("nan")
    got = packed_attention(q, k, v, plan)
    assert torch.equal(got[:6], clean[:6]) and got[6, 0, 2] == float("inf") and got[8:].isnan().all()


def test_host_adapters():
    ids, lens = [1, -1, 0, 1], [3, 4, 0, 6]
    x, y = rnd(1, 13, 24).to(HF), rnd(2, 13, 10).to(HF)
    down, up, scale = rnd(3, 2, 8, 24).to(HF), rnd(4, 2, 10, 8).to(HF), torch.tensor([0.5, 2.0])
    plan = AdapterPlan(ids, lens, adapters=2, device="cpu")
    ref = U.adapters(y, x, down, up, ids, lens, scale)
    U.check(adapter_add(y, x, down, up, plan, scale=scale), *ref)
    assert adapter_add(y, x, down, up, plan, scale=scale, out=y) is y
    U.check(y, *ref)


# -------------------------------------------------------------------------------------------------------------- module

def make_block(dim=64, heads=4, kv_heads=2, head_dim=16, group=16, adapters=2, device="cpu"):
    from hyperflow_h3_flash_amd import AttentionBlock

    block = AttentionBlock(dim, heads, head_dim, group, kv_heads=kv_heads, adapters=adapters, adapter_rank=5)
    gen = torch.Generator().manual_seed(2)
    for layer in (block.qkv, block.out):
        layer.qweight.copy_(torch.randint(-127, 128, layer.qweight.shape, generator=gen, dtype=torch.int8))
        layer.wscale.copy_(0.02 * torch.rand(layer.wscale.shape, generator=gen) / layer.in_features ** 0.5)
    block.norm_q.copy_(1 + 0.1 * torch.randn(head_dim, generator=gen))
    block.norm_k.copy_(1 + 0.1 * torch.randn(head_dim, generator=gen))
    for bank in (block.qkv_adapters, block.out_adapters) if adapters else ():
        for i in range(adapters):
            bank.load(i, torch.randn(5, bank.in_features, generator=gen), torch.randn(bank.out_features, 5, generator=gen),
                      scale=0.1 + i)
    return block.to(device)


def test_block_is_its_parts_and_requests_stay_alone():
    from hyperflow_h3_flash_amd import AttentionBlock, Int8RotLinear

    block = make_block()
    lengths, ids = [5, 9, 1], [1, -1, 0]
    x = rnd(1, 15, 64).to(BF)
    positions = torch.randint(0, 50, (15, 2), generator=torch.Generator().manual_seed(3))
    rotary = RotaryAxes((8, 8))

    def run(rows, lengths, ids, module=block):
        plan = AttentionPlan(lengths, heads=4, kv_heads=2, head_dim=16, causal=True, device="cpu")
        adapters = AdapterPlan(ids, lengths, adapters=2, device="cpu") if module.qkv_adapters is not None else None
        return module(x[rows], plan, positions=positions[rows], rotary=rotary, adapters=adapters)

    whole = run(slice(0, 15), lengths, ids)
    assert whole.shape == (15, 64) and whole.dtype is BF
    at = 0
    for n, i in zip(lengths, ids):
        assert torch.equal(run(slice(at, at + n), [n], [i]), whole[at:at + n])
        at += n
    # the parts by hand
    qkv = block.qkv(x)
    plan = AdapterPlan(ids, lengths, adapters=2, device="cpu")
    qkv = block.qkv_adapters(qkv, x, plan).view(15, 8, 16)
    q, k = qk_norm_rope(qkv[:, :4], qkv[:, 4:6], positions, rotary, q_weight=block.norm_q, k_weight=block.norm_k)
    o = packed_attention(q, k, qkv[:, 6:], AttentionPlan(lengths, heads=4, kv_heads=2, head_dim=16, causal=True,
                                                         device="cpu")).reshape(15, 64)
    assert torch.equal(block.out_adapters(block.out(o), o, plan), whole)
    # from a model's own projections
    layers = [Int8RotLinear(64, n, 16) for n in (64, 32, 32)]
    for layer, rows in zip(layers, (slice(0, 64), slice(64, 96), slice(96, 128))):
        layer.qweight.copy_(block.qkv.qweight[rows])
        layer.wscale.copy_(block.qkv.wscale[rows])
    again = AttentionBlock.from_projections(*layers, block.out, 16)
    assert again.kv_heads == 2 and not any(p.requires_grad or p.is_meta for p in again.parameters())
    plain = make_block(adapters=0)
    plain.norm_q.fill_(1)
    plain.norm_k.fill_(1)
    assert torch.equal(run(slice(0, 15), lengths, ids, again), run(slice(0, 15), lengths, ids, plain))
    banked = AttentionBlock.from_projections(*layers, block.out, 16, adapters=2, adapter_rank=8)
    assert torch.equal(run(slice(0, 15), lengths, ids, banked), run(slice(0, 15), lengths, ids, plain))


def test_refusals_of_the_block():
    from hyperflow_h3_flash_amd import AdapterBank, AttentionBlock, Int8RotLinear

    bank = AdapterBank(32, 16, 2, 5)
    assert bank.rank == 8
    for bad in (
        lambda: AdapterBank(32, 16, 0, 8), lambda: AdapterBank(32, 16, 2, 0),
        lambda: bank.load(2, torch.zeros(4, 32), torch.zeros(16, 4)),
        lambda: bank.load(0, torch.zeros(9, 32), torch.zeros(16, 9)),
        lambda: bank.load(0, torch.zeros(4, 32), torch.zeros(16, 5)),
        lambda: make_block(adapters=0)(rnd(1, 3, 64).to(BF), AttentionPlan([3], heads=4, kv_heads=2, head_dim=16,
                                                                          device="cpu"),
                                       adapters=AdapterPlan([0], [3], adapters=1, device="cpu")),
        lambda: AttentionBlock.from_projections(*(Int8RotLinear(64, n, 16) for n in (64, 32, 64)),
                                                Int8RotLinear(64, 64, 16), 16),
        lambda: AttentionBlock.from_projections(*(Int8RotLinear(64, 64, 16) for _ in range(3)),
                                                Int8RotLinear(32, 64, 16), 16),
    ):
        with pytest.raises(ValueError):
            bad()


def test_example_runs_on_the_host():
    import importlib.util

    spec = importlib.util.spec_from_file_location("example", os.path.join(_native.REPO_DIR, "examples",
                                                                          "packed_attention_block.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    y = example.main(requests=((2, 2, 3), (1, 2, 2), (1, 1, 1)), dim=256, heads=2, device="cpu")
    assert y.shape == (17, 256) and y.isfinite().all()


# ----------------------------------------------------------------------------------------------------------- refusals

def test_refusals_of_the_norm_and_rotation():
    q, k = rnd(1, 4, 2, 64).to(BF), rnd(2, 4, 2, 64).to(BF)
    p, r = torch.arange(4), RotaryAxes((64,))
    for bad in (
        lambda: RotaryAxes(()), lambda: RotaryAxes((15, 17)), lambda: RotaryAxes((8,)), lambda: RotaryAxes((16, -16)),
        lambda: RotaryAxes((16,), theta=0.0), lambda: RotaryAxes((16,), theta=float("inf")),
        lambda: qk_norm_rope(q[0], None, p, r), lambda: qk_norm_rope(q, k[:3], p, r),
        lambda: qk_norm_rope(q, k[..., :32], p, r), lambda: qk_norm_rope(q, k.to(HF), p, r),
        lambda: qk_norm_rope(q.float(), None, p, r), lambda: qk_norm_rope(q[..., :40], None, p, r),
        lambda: qk_norm_rope(q[..., :32], None, p, r), lambda: qk_norm_rope(q, None, p[:3], r),
        lambda: qk_norm_rope(q, None, p.to(torch.int16), r), lambda: qk_norm_rope(q, None, None, r),
        lambda: qk_norm_rope(q, None, p, RotaryAxes((32, 32))), lambda: qk_norm_rope(q, None, p, r, eps=-1.0),
        lambda: qk_norm_rope(q, None, p, r, eps=float("nan")),
        lambda: qk_norm_rope(q, None, p, r, q_weight=torch.ones(32)),
        lambda: qk_norm_rope(q, None, p, r, q_weight=torch.ones(64), norm=False),
        lambda: qk_norm_rope(q, None, p, r, out=(q[:2], None)), lambda: qk_norm_rope(q, k, p, r, out=(q, k.to(HF))),
    ):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="forward only"):
        qk_norm_rope(q.clone().requires_grad_(), None, p, r)
    with torch.no_grad():
        qk_norm_rope(q.clone().requires_grad_(), None, p, r)


def test_refusals_of_attention():
    def plan(q=(4,), kv=None, heads=2, kv_heads=2, head_dim=32, **more):
        return AttentionPlan(q, kv, heads=heads, kv_heads=kv_heads, head_dim=head_dim, device="cpu", **more)

    q = rnd(1, 4, 2, 32).to(BF)
    p = plan()
    for bad in (
        lambda: plan(q=(-1,)), lambda: plan(kv=(1, 2)), lambda: plan(heads=3), lambda: plan(heads=0),
        lambda: plan(kv_heads=0), lambda: plan(head_dim=24), lambda: plan(head_dim=144), lambda: plan(head_dim=0),
        lambda: packed_attention(q[:3], q, q, p), lambda: packed_attention(q, q[:3], q, p),
        lambda: packed_attention(q, q, q[:, :1], p), lambda: packed_attention(q, q.to(HF), q, p),
        lambda: packed_attention(q.float(), q.float(), q.float(), p), lambda: packed_attention(q, q, q, p, scale=0.0),
        lambda: packed_attention(q, q, q, p, scale=-1.0), lambda: packed_attention(q, q, q, p, scale=float("nan")),
        lambda: packed_attention(q, q, q, p, out=q.float()),
    ):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="forward only"):
        packed_attention(q, q, q.clone().requires_grad_(), p)


def test_refusals_of_adapters():
    x, y = rnd(1, 4, 16).to(BF), rnd(2, 4, 6).to(BF)
    down, up = rnd(3, 2, 8, 16).to(BF), rnd(4, 2, 6, 8).to(BF)
    plan = AdapterPlan([0, 1], [2, 2], adapters=2, device="cpu")
    for bad in (
        lambda: AdapterPlan([2], adapters=2, device="cpu"), lambda: AdapterPlan([-2], adapters=2, device="cpu"),
        lambda: AdapterPlan([0], [1, 2], adapters=2, device="cpu"),
        lambda: AdapterPlan([0], [-1], adapters=2, device="cpu"),
        lambda: adapter_add(y, x[:3], down, up, plan), lambda: adapter_add(y[:3], x, down, up, plan),
        lambda: adapter_add(y, x, down[:1], up, plan), lambda: adapter_add(y, x, down, up[:, :5], plan),
        lambda: adapter_add(y, x, down[:, :4], up[..., :4], plan),
        lambda: adapter_add(y, x[:, :12], down[..., :12], up, plan), lambda: adapter_add(y, x.to(HF), down, up, plan),
        lambda: adapter_add(*(t.float() for t in (y, x, down, up)), plan),
        lambda: adapter_add(y, x, down, up, plan, scale=torch.ones(3)),
        lambda: adapter_add(y, x, down, up, plan, scale=torch.ones(2, dtype=BF)),
        lambda: adapter_add(y, x, down, up, plan, out=y[:2]),
    ):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="forward only"):
        adapter_add(y, x, down.clone().requires_grad_(), up, plan)


# -------------------------------------------------------------------------------------------------------------- C ABI

def test_header_and_binding_agree(lib):
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = re.findall(r"^\s*(?:const\s+)?\w+\s*\*?\s*(hf_\w+)\s*\(", text, flags=re.M)
    assert sorted(names) == sorted(_native.BLOCK_SIGNATURES)
    for name, (args, _) in _native.BLOCK_SIGNATURES.items():
        assert hasattr(lib, name)
        declared = re.search(name + r"\s*\((.*?)\)", text, flags=re.S).group(1)
        assert len(declared.split(",")) == len(args), name


def attention_plan(lib, q, kv, heads=2, kv_heads=1, D=64, causal=0, cus=256):
    qa, ka = (ctypes.c_int64 * max(len(q), 1))(*q), (ctypes.c_int64 * max(len(kv), 1))(*kv)
    n = lib.hf_attention_plan(qa, ka, len(q), heads, kv_heads, D, causal, cus, None, 0)
    if n < 0:
        return n
    buf = ctypes.create_string_buffer(n)
    assert lib.hf_attention_plan(qa, ka, len(q), heads, kv_heads, D, causal, cus, buf, n - 1) == -5
    assert lib.hf_attention_plan(qa, ka, len(q), heads, kv_heads, D, causal, cus, buf, n) == n
    return buf


def test_argument_checks_reject_before_launching(lib):
    fake, odd = ctypes.c_void_p(1 << 20), ctypes.c_void_p((1 << 20) + 2)

    def rope(q=fake, token=128, heads=2, heads_k=0, out=fake, pos=fake, pos_type=0, ld=1, axes=1, turns=fake, pairs=32,
             eps=1e-6, T=4, D=64, dtype=0, qw=None, k=None):
        return lib.hf_qk_norm_rope(q, token, 64, heads, k, 64, 64, heads_k, out, token, 64, None, 64, 64, pos, pos_type,
                                   ld, axes, turns, turns, pairs, 1, 1, qw, None, 0, eps, T, D, dtype, None)

    assert rope(T=0) == 0
    assert rope(q=None) == rope(out=None) == rope(pos=None) == rope(turns=None) == -1
    assert rope(T=-1) == rope(dtype=2) == rope(pos_type=3) == rope(eps=-1.0) == rope(axes=0) == rope(heads_k=1) == -1
    assert rope(pairs=40) == -1 and rope(axes=2) == -1
    assert rope(D=72) == rope(pairs=12) == rope(q=odd) == rope(token=130) == rope(qw=odd) == -3
    assert rope(T=1 << 31) == rope(D=272) == rope(axes=17, ld=17) == rope(heads=70000) == -5

    plan = attention_plan(lib, [5], [700])
    n = len(plan.raw)

    def attend(q=fake, k=fake, tok=128, head=64, scale=0.1, plan=plan, dev=fake, bytes_=n, ws=fake, ws_bytes=1 << 30,
               dtype=0):
        return lib.hf_attention(q, tok, head, k, tok, head, k, tok, head, q, tok, head, scale, plan, dev, bytes_, ws,
                                ws_bytes, dtype, None)

    assert lib.hf_attention_ws_bytes(plan, n) > 0 and lib.hf_attention_ws_bytes(plan, n - 4) == -1
    assert lib.hf_attention_ws_bytes(None, 0) == -1
    assert attend(q=None) == attend(k=None) == attend(dev=None) == attend(plan=None) == attend(bytes_=n + 1) == -1
    assert attend(scale=0.0) == attend(scale=float("nan")) == attend(dtype=7) == attend(tok=-8) == -1
    assert attend(tok=32) == -1  # rows of keys that overlap
    assert attend(ws=None) == attend(ws_bytes=16) == -1
    assert attend(q=odd) == attend(k=odd) == attend(head=60) == attend(dev=odd) == -3
    assert attend(tok=1 << 23) == -5
    empty = attention_plan(lib, [0], [5])
    assert attend(q=None, k=None, plan=empty, bytes_=len(empty.raw)) == 0
    assert attention_plan(lib, [-1], [5]) == attention_plan(lib, [1], [-5]) == -1
    assert attention_plan(lib, [1], [5], heads=3, kv_heads=2) == attention_plan(lib, [1], [5], heads=0) == -1
    assert attention_plan(lib, [1], [5], D=72) == -3 and attention_plan(lib, [1], [5], D=144) == -5
    assert attention_plan(lib, [1 << 31], [5]) == attention_plan(lib, [1 << 30, 1 << 30], [5, 5]) == -5

    ids, lens = (ctypes.c_int32 * 2)(0, -1), (ctypes.c_int64 * 2)(40, 3)
    size = lib.hf_adapter_plan(ids, lens, 2, 1, 256, None, 0)
    buf = ctypes.create_string_buffer(size)
    assert lib.hf_adapter_plan(ids, lens, 2, 1, 256, buf, size - 1) == -5
    assert lib.hf_adapter_plan(ids, lens, 2, 1, 256, buf, size) == size
    assert lib.hf_adapter_plan(ids, lens, 2, 0, 256, None, 0) == -1  # adapter 0 of none
    assert lib.hf_adapter_plan((ctypes.c_int32 * 1)(-2), None, 1, 3, 256, None, 0) == -1
    assert lib.hf_adapter_plan(ids, (ctypes.c_int64 * 2)(1 << 31, 1), 2, 1, 256, None, 0) == -5
    need = lib.hf_adapter_ws_bytes(buf, size, 512, 24, 1)
    assert need >= 40 * 32 * 4
    assert lib.hf_adapter_ws_bytes(buf, size - 1, 512, 24, 1) == lib.hf_adapter_ws_bytes(buf, size, 512, 520, 1) == -1
    assert lib.hf_adapter_ws_bytes(buf, size, 512, 24, 2) == -1

    def adapt(x=fake, ldx=512, y=fake, ldy=64, down=fake, r=24, out=fake, ldo=64, N=64, K=512, plan=buf, dev=fake,
              ws=fake, ws_bytes=need, dtype=1):
        return lib.hf_adapter_add(x, ldx, y, ldy, down, down, r, None, out, ldo, N, K, plan, dev, size, ws, ws_bytes,
                                  dtype, None)

    assert adapt(N=0) == 0
    assert adapt(x=None) == adapt(y=None) == adapt(down=None) == adapt(out=None) == adapt(dev=None) == -1
    assert adapt(plan=None) == adapt(dtype=2) == adapt(ldx=504) == adapt(ldy=63) == adapt(K=0) == adapt(r=0) == -1
    assert adapt(ws=None) == adapt(ws_bytes=need - 1) == adapt(ldo=72) == -1  # in place with another stride
    assert adapt(K=508) == adapt(r=12) == adapt(ldx=516) == adapt(x=odd) == adapt(down=odd) == -3
    assert adapt(r=520) == -5


@pytest.mark.parametrize("name,packer", [("hf_qk_norm_rope", _native.ROPE_ARGS), ("hf_attention", _native.ATTENTION_ARGS),
                                         ("hf_adapter_add", _native.ADAPTER_ARGS)])
def test_structs_hold_the_parameters_in_their_order(name, packer):
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    declared = [" ".join(p.split()) for p in re.search(r"int " + name + r"\((.*?)\)", text, flags=re.S).group(1).split(",")]
    body = re.search(r"typedef struct \{([^}]*)\} " + name + "_args;", text).group(1)
    assert [" ".join(p.split()) for p in body.split(";")[:-1]] == declared
    kinds = {"int64_t": "q", "int32_t": "i", "float": "f"}
    assert packer.format == "@" + "".join(kinds.get(p.rsplit(" ", 1)[0], "P") for p in declared)
    assert packer.size % struct.calcsize("P") == 0


def test_calls_by_struct_refuse_as_the_lists_do(lib):
    rope = [1 << 20, 128, 64, 2, 0, 64, 64, 0, 1 << 20, 128, 64, 0, 64, 64, 1 << 20, 0, 1, 1, 1 << 20, 1 << 20, 32, 1, 1,
            0, 0, 0, 1e-6, 0, 64, 0, 0]
    assert lib.hf_qk_norm_rope_call(_native.ROPE_ARGS.pack(*rope)) == 0  # no tokens
    for at, value, status in ((0, 0, -1), (8, 0, -1), (28, 72, -3), (29, 2, -1), (27, 1 << 31, -5), (1, 130, -3)):
        assert lib.hf_qk_norm_rope_call(_native.ROPE_ARGS.pack(*(
            value if i == at else 4 if i == 27 else x for i, x in enumerate(rope)))) == status, at
    plan = attention_plan(lib, [0], [5])
    attend = [0, 128, 64, 0, 128, 64, 0, 128, 64, 0, 128, 64, 0.1, ctypes.addressof(plan), 0, len(plan.raw), 0, 0, 0, 0]
    assert lib.hf_attention_call(_native.ATTENTION_ARGS.pack(*attend)) == 0  # no queries
    for at, value in ((12, 0.0), (15, len(plan.raw) + 4), (18, 7)):
        assert lib.hf_attention_call(_native.ATTENTION_ARGS.pack(*(
            value if i == at else x for i, x in enumerate(attend)))) == -1, at
    ids = (ctypes.c_int32 * 1)(0)
    size = lib.hf_adapter_plan(ids, None, 1, 1, 256, None, 0)
    buf = ctypes.create_string_buffer(size)
    assert lib.hf_adapter_plan(ids, None, 1, 1, 256, buf, size) == size
    adapt = [1 << 20, 512, 1 << 20, 64, 1 << 20, 1 << 20, 24, 0, 1 << 20, 64, 0, 512, ctypes.addressof(buf), 1 << 20, size,
             0, 0, 1, 0]
    assert lib.hf_adapter_add_call(_native.ADAPTER_ARGS.pack(*adapt)) == 0  # no columns
    for at, value, status in ((6, 0, -1), (6, 520, -5), (11, 508, -3), (14, size + 1, -1), (17, 2, -1)):
        assert lib.hf_adapter_add_call(_native.ADAPTER_ARGS.pack(*(
            value if i == at else x for i, x in enumerate(adapt)))) == status, at
    assert (lib.hf_qk_norm_rope_call(None) == lib.hf_attention_call(None) == lib.hf_adapter_add_call(None) == -1)


def test_planners_refuse_sizes_that_their_memory_would_go_with(lib):
    one, ids = (ctypes.c_int64 * 1)(5), (ctypes.c_int32 * 1)(0)
    assert lib.hf_attention_plan(one, one, 1, 2, 1, 64, 0, 65537, None, 0) == -1
    assert lib.hf_attention_plan(one, one, 1, 2, 1, 64, 0, 65536, None, 0) > 0
    assert lib.hf_adapter_plan(ids, None, 1, 1, 65537, None, 0) == -1
    assert lib.hf_adapter_plan(ids, None, 1, (1 << 24) + 1, 256, None, 0) == -5


# ----------------------------------------------------------------------------------------------------------- planners

@pytest.mark.parametrize("q,kv,heads,kv_heads,causal", [
    ([37710], [37710], 7, 7, 0), ([5, 0, 300, 1], [5, 9, 300, 4000], 8, 2, 1), ([1] * 16, list(range(1, 16001, 1000)), 32, 8, 1),
    ([130, 40], [0, 50000], 4, 1, 0), ([900, 3], [100, 700], 6, 3, 1), ([], [], 2, 1, 0), ([64] * 40, [64] * 40, 1, 1, 1), ([3, 200], [0, 0], 2, 1, 0),
    ([4099, 1537, 300, 61, 2048], [4099, 1537, 300, 61, 2048], 32, 8, 1),
])
def test_attention_plan_covers_every_row_and_key_once(lib, q, kv, heads, kv_heads, causal):
    raw = attention_plan(lib, q, kv, heads, kv_heads, 64, causal).raw
    *_, items, joins, _ = struct.unpack_from("8i", raw)
    rows = 128
    size, slots, q_rows, kv_rows = struct.unpack_from("4q", raw, 32)
    assert size == len(raw) and (q_rows, kv_rows) == (sum(q), sum(kv))
    item = np.frombuffer(raw, np.int32, items * 12, 128).reshape(items, 12)
    join = np.frombuffer(raw, np.int32, joins * 8, 128 + items * 48).reshape(joins, 8)
    group = heads // kv_heads
    tiles = {}
    for q0, nq, k0, nk, row0, lo, hi, head, slot, *_ in item.tolist():
        assert 0 <= lo <= hi <= nk and lo % 64 == 0 and row0 % rows == 0
        tiles.setdefault((q0, nq, k0, nk, row0, head), []).append((lo, hi, slot))
    shares = {(q0, nq, k0, nk, row0, head): (first, n) for q0, nq, k0, nk, row0, head, first, n in join.tolist()}
    want, used, q0, k0 = set(), [], 0, 0
    for nq, nk in zip(q, kv):
        for row0 in range(0, nq * group, rows):
            last = min(row0 + rows, nq * group) - 1
            need = min(max(last // group + nk - nq + 1, 0), nk) if causal else nk
            for head in range(kv_heads):
                key = (q0, nq, k0, nk, row0, head)
                want.add(key)
                parts = sorted(tiles[key])
                assert parts[0][0] == 0 and parts[-1][1] == need
                assert all(a[1] == b[0] for a, b in zip(parts, parts[1:]))
                if len(parts) == 1:
                    assert parts[0][2] == -1 and key not in shares
                else:
                    first, n = shares.pop(key)
                    assert sorted(p[2] for p in parts) == list(range(first, first + n))
                    used += range(first, first + n)
        q0, k0 = q0 + nq, k0 + nk
    assert want == set(tiles) and not shares and sorted(used) == list(range(slots))


@pytest.mark.parametrize("cus", [1, 256])
@pytest.mark.parametrize("ids,lens", [([0, 2, -1, 0], [70, 1, 5, 3]), ([-1], [9]), ([], []), ([1] * 200, None),
                                      ([2, 1, 0, 1, 2, -1], [0, 64, 65, 1, 200, 64])])
def test_adapter_plan_covers_every_row_once(lib, ids, lens, cus):
    n = [1] * len(ids) if lens is None else lens
    ids_c = (ctypes.c_int32 * max(len(ids), 1))(*ids)
    lens_c = None if lens is None else (ctypes.c_int64 * max(len(ids), 1))(*lens)
    size = lib.hf_adapter_plan(ids_c, lens_c, len(ids), 3, cus, None, 0)
    buf = ctypes.create_string_buffer(size)
    assert lib.hf_adapter_plan(ids_c, lens_c, len(ids), 3, cus, buf, size) == size
    _, adapters, tiles, live = struct.unpack_from("4i", buf.raw)
    _, rows, live_rows, tile_rows = struct.unpack_from("3qi", buf.raw, 16)
    assert tile_rows in (32, 64) and (tile_rows == 32 or cus == 1)
    of = [a for a, c in zip(ids, n) for _ in range(c)]
    assert (adapters, rows, live_rows) == (3, len(of), sum(a >= 0 for a in of))
    tile = np.frombuffer(buf.raw, np.int32, tiles * 4, 128).reshape(tiles, 4)
    order = np.frombuffer(buf.raw, np.int32, rows, 128 + 16 * tiles)
    assert sorted(order.tolist()) == list(range(rows))
    at = 0
    for i, (a, start, count, _) in enumerate(tile.tolist()):
        assert start == at and 1 <= count <= tile_rows and (a >= 0) == (i < live)
        assert all(of[r] == a for r in order[start:start + count])
        assert (np.diff(order[start:start + count]) > 0).all()
        at += count
    assert at == rows

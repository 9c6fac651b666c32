"""Transformer blocks around the INT8 linears: equal to their parts, a step over the cache to the whole, and refusals; on the
host, and on the GPU."""

from __future__ import annotations

import os
import sys

import pytest
import torch

from hyperflow_h3_flash_amd import (AttentionPlan, Int8RotLinear, KVCache, RotaryAxes, RowPlan, TransformerBlock,
                                    TransformerStack, _native, residual_norm)
from test_block import make_block

BF = torch.bfloat16
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def rnd(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def int8(k, n, group, seed, **kw):
    layer = Int8RotLinear(k, n, group, **kw)
    gen = torch.Generator().manual_seed(seed)
    layer.qweight.copy_(torch.randint(-127, 128, layer.qweight.shape, generator=gen, dtype=torch.int8))
    layer.wscale.fill_(k ** -0.5 / 73)
    return layer


def make(seed, device, dim=64, heads=4, kv_heads=2, head_dim=16, group=16, inner=96, **kw):
    attention = make_block(dim=dim, heads=heads, kv_heads=kv_heads, head_dim=head_dim, group=group, adapters=0)
    block = TransformerBlock(attention, int8(dim, 2 * inner, group, seed, activation="swiglu"), int8(inner, dim, group, seed + 1),
                             **kw)
    for i, name in enumerate(("norm_attention", "norm_ff", "post_attention", "post_ff")):
        if getattr(block, name) is not None:
            getattr(block, name).copy_(1 + 0.1 * rnd(seed + 2 + i, dim))
    return block.to(device)


SIZES = {"cpu": {}, "cuda": dict(dim=512, heads=8, kv_heads=2, head_dim=64, group=256, inner=768)}


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("norm,post,stream", [("layer", None, BF), ("rms", "rms", torch.float32)])
def test_a_stack_is_its_parts(device, norm, post, stream):
    size = SIZES[device]
    blocks = [make(10 * i, device, norm=norm, post_norm=post, **size) for i in range(2)]
    dim, D = blocks[0].dim, size.get("head_dim", 16)
    heads, kv_heads = size.get("heads", 4), size.get("kv_heads", 2)
    lengths = [5, 9, 1]
    x = rnd(1, 15, dim).to(stream).to(device)
    m = [(0.3 * rnd(2 + i, 3, 6, dim)).to(BF).to(device) for i in range(2)]
    rows = RowPlan(lengths, device=device)
    rotary, positions = RotaryAxes((16,)), torch.arange(15, device=device)
    plan = AttentionPlan(lengths, heads=heads, kv_heads=kv_heads, head_dim=D, device=device)
    got = TransformerStack(blocks)(x, plan, modulation=m, rows=rows, positions=positions, rotary=rotary)
    assert got.shape == x.shape and got.dtype is stream
    want = x
    for block, mod in zip(blocks, m):
        shift, scale, gate, shift2, scale2, gate2 = (mod[:, i] for i in range(6))
        n = residual_norm(want, rows=rows, norm=norm, weight=block.norm_attention, scale=scale, shift=shift)[1]
        a = block.attention(n, plan, positions=positions, rotary=rotary)
        want, n = residual_norm(want, a, rows=rows, gate=gate, post_norm=post, post_weight=block.post_attention, norm=norm,
                                weight=block.norm_ff, scale=scale2, shift=shift2)
        want, _ = residual_norm(want, block.down(block.up(n)), rows=rows, gate=gate2, post_norm=post,
                                post_weight=block.post_ff, norm=None)
    # The stack takes the second block's first norm from a stream that is not rounded in between, the parts from the rounded
    # one: inputs of the INT8 layers differ in their last bit, and codes with them.
    first = blocks[0](x, plan, modulation=m[0], rows=rows, positions=positions, rotary=rotary)
    alone = TransformerStack(blocks[:1])(x, plan, modulation=m[:1], rows=rows, positions=positions, rotary=rotary)
    assert torch.equal(first, alone)
    assert (got - want).float().norm() <= 0.05 * want.float().norm()
    plain = TransformerStack([make(0, device, norm=norm, weights=False, **size)])(x, plan)  # neither modulation nor weights
    assert plain.isfinite().all() and not torch.equal(plain, x)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("stream", [BF, torch.float32])
@pytest.mark.parametrize("eps", [(1e-6, 1.0), (1.0, 1e-6)])
def test_each_block_of_a_stack_keeps_its_eps(device, stream, eps):
    """The norm behind a block's feed-forward has that block's eps, the one before the next block's attention the next
    block's. The blocks one by one round the stream in the same place, so the results are the same bits."""
    size = SIZES[device]
    blocks = [make(10 * i, device, norm="rms", post_norm="rms", eps=e, **size) for i, e in enumerate(eps)]
    x = (0.5 * rnd(1, 15, blocks[0].dim)).to(stream).to(device)
    plan = AttentionPlan([5, 9, 1], heads=size.get("heads", 4), kv_heads=size.get("kv_heads", 2),
                         head_dim=size.get("head_dim", 16), device=device)
    m = [(0.3 * rnd(2 + i, 3, 6, blocks[0].dim)).to(BF).to(device) for i in range(2)]
    rows = RowPlan([5, 9, 1], device=device)
    want = x
    for block, mod in zip(blocks, m):
        want = block(want, plan, modulation=mod, rows=rows)
    assert torch.equal(TransformerStack(blocks)(x, plan, modulation=m, rows=rows), want)


@pytest.mark.parametrize("device", DEVICES)
def test_steps_over_the_cache_agree_with_each_other(device):
    """A prompt in one step, in two, and its last token alone give the same last rows; a fork does not change its source."""
    size = SIZES[device]
    stack = TransformerStack([make(10 * i, device, norm="rms", **size) for i in range(2)])
    dim, D, heads, kv_heads = stack.blocks[0].dim, size.get("head_dim", 16), size.get("heads", 4), size.get("kv_heads", 2)
    n = 40
    x = rnd(3, n, dim).to(BF).to(device)
    rotary, positions = RotaryAxes((16,)), torch.arange(n, device=device)

    def run(cache, request, lo, hi):
        plan = cache.plan([request], [hi - lo], heads=heads, causal=True)
        return stack(x[lo:hi], plan, positions=positions[lo:hi], rotary=rotary)

    cache = KVCache(2, kv_heads, D, 12, page_size=32, device=device)
    whole = run(cache, cache.new(), 0, n)
    b = cache.new()
    parts = [run(cache, b, 0, 33)]
    c = cache.fork(b)
    parts.append(run(cache, b, 33, n - 1))
    parts.append(run(cache, b, n - 1, n))
    fork = run(cache, c, 33, n)
    # The same rows in other tiles: sums in another order, whose last bits INT8 codes may turn into a step.
    parts = torch.cat(parts)
    for got, want in ((parts, whole), (fork, whole[33:])):
        assert (got - want).float().norm() <= 0.02 * want.float().norm()
    assert cache.length(c) == n and cache.table(b)[1] != cache.table(c)[1]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("to", [torch.float16, torch.float32])
def test_a_converted_block_keeps_working(device, to):
    """Weights that every type holds (one, quarters), after `Module.to`: the same bits."""
    size = SIZES[device]
    blocks = [make(10 * i, device, norm="rms", post_norm="rms", **size) for i in range(2)]
    for block in blocks:
        for name in ("norm_attention", "norm_ff", "post_attention", "post_ff"):
            getattr(block, name).copy_(1 + torch.arange(block.dim) % 3 / 4)
        for w in (block.attention.norm_q, block.attention.norm_k):
            w.fill_(1.25)
    plan = AttentionPlan([7], heads=size.get("heads", 4), kv_heads=size.get("kv_heads", 2), head_dim=size.get("head_dim", 16),
                         device=device)
    stack = TransformerStack(blocks)
    for layer in stack.modules():  # scales of the INT8 layers that float16 holds too
        if isinstance(layer, Int8RotLinear):
            layer.wscale.fill_(2.0 ** -9)
    x = rnd(1, 7, blocks[0].dim).to(BF).to(device)
    want = stack(x, plan)
    assert torch.equal(stack.to(to)(x, plan), want)


def test_refusals_of_the_blocks():
    block = make(0, "cpu")
    x, plan = rnd(1, 3, 64).to(BF), AttentionPlan([3], heads=4, kv_heads=2, head_dim=16, device="cpu")
    m = torch.zeros(1, 6, 64, dtype=BF)
    cache = KVCache(1, 2, 16, 4, device="cpu")
    step = cache.plan([cache.new()], [3], new_lengths=[2], heads=4)
    for bad in (lambda: TransformerBlock(block.attention, block.down, block.down),
                lambda: TransformerBlock(block.attention, block.up, block.up),
                lambda: TransformerBlock(block.attention, block.up, block.down, norm="batch"),
                lambda: TransformerBlock(block.attention, block.up, block.down, norm=None),
                lambda: TransformerStack([block, make(0, "cpu", dim=32, heads=2, kv_heads=1)]),
                lambda: block(x, plan, modulation=m[:, :5]), lambda: block(x, plan, modulation=m.expand(2, 6, 64)),
                lambda: TransformerStack([block])(x, plan, modulation=[m, m]), lambda: block(x, step)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="forward only"):
        block(x.clone().requires_grad_(), plan)
    assert TransformerStack([])(x, plan) is x


@pytest.mark.parametrize("device", DEVICES)
def test_example_runs(device):
    sys.path.insert(0, os.path.join(_native.REPO_DIR, "examples"))
    import cached_transformer_block

    small = dict(dim=64, heads=2, head_dim=32, inner=64, group=16) if device == "cpu" else {}
    out = cached_transformer_block.main(chunk=(1, 3, 5), chunks=3, device=device, **small)
    assert out.shape[0] == 2 * 15 and out.isfinite().all()

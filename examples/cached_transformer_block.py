"""A clip extended chunk by chunk through transformer blocks over a 4-bit cache: `python examples/cached_transformer_block.py`.

Random weights: two blocks of eight heads of 128 on the reference model's token width, 5376. Each chunk's latent frames attend
to all earlier ones, whose keys and values are held in 4 bits; before the last chunk the clip is forked, and the two
continuations share the pages of what they have in common."""

from __future__ import annotations

import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from hyperflow_h3_flash_amd import (AttentionBlock, Int8RotLinear, KVCache, RotaryAxes, RowPlan, TransformerBlock,  # noqa: E402
                                    TransformerStack)


def fill(layer: Int8RotLinear, gen: torch.Generator) -> Int8RotLinear:
    layer.qweight.copy_(torch.randint(-127, 128, layer.qweight.shape, generator=gen, dtype=torch.int8))
    layer.wscale.fill_(layer.in_features ** -0.5 / 73)
    return layer


def main(chunk=(3, 30, 54), chunks=3, dim=5376, heads=8, head_dim=128, inner=7168, group=256, blocks=2,
         device=None) -> torch.Tensor:
    device = device or ("cuda" if torch.cuda.is_available() else "cpu")
    gen = torch.Generator().manual_seed(0)
    stack = []
    for _ in range(blocks):
        attention = AttentionBlock(dim, heads, head_dim, group)
        fill(attention.qkv, gen), fill(attention.out, gen)
        stack.append(TransformerBlock(attention, fill(Int8RotLinear(dim, 2 * inner, group, activation="swiglu"), gen),
                                      fill(Int8RotLinear(inner, dim, group), gen), norm="layer", weights=False))
    model = TransformerStack(stack).to(device)
    n = chunk[0] * chunk[1] * chunk[2]
    cache = KVCache(blocks, heads, head_dim, pages=-(-(chunks + 1) * n // 64) + 2, device=device)
    rotary = RotaryAxes((head_dim // 2, head_dim // 4, head_dim // 4), device=device)
    grid = torch.cartesian_prod(*(torch.arange(c) for c in chunk)).int()

    clips = [cache.new()]
    for i in range(chunks):
        if i == chunks - 1:
            clips.append(cache.fork(clips[0]))
        lengths = [n] * len(clips)
        plan = cache.plan(clips, lengths, heads=heads)
        rows = RowPlan(lengths, device=device)
        positions = (grid + torch.tensor([i * chunk[0], 0, 0], dtype=torch.int32)).repeat(len(clips), 1).to(device)
        x = torch.randn(sum(lengths), dim, generator=gen).to(torch.bfloat16).to(device)
        modulation = [(0.1 * torch.randn(len(clips), 6, dim, generator=gen)).to(torch.bfloat16).to(device) for _ in range(blocks)]
        began = time.perf_counter()
        y = model(x, plan, modulation=modulation, rows=rows, positions=positions, rotary=rotary)
        if y.is_cuda:
            torch.cuda.synchronize()
            print(f"chunk {i}: {sum(lengths)} new tokens, {sum(plan.kv_lengths)} cached: "
                  f"{(time.perf_counter() - began) * 1e3:.2f} ms, {cache.free_pages} pages free")
    return y


if __name__ == "__main__":
    print(main().shape)

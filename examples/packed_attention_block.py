"""Three video requests of different sizes through one attention block: `python examples/packed_attention_block.py`.

Random weights: eight heads of 128 on the reference model's token width, 5376. The requests' tokens lie one behind the other; each attends within itself, turned by its own (time, height,
width) positions, and takes its own adapter. The plans depend on lengths and requests alone and serve every layer and
step."""

from __future__ import annotations

import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from hyperflow_h3_flash_amd import AdapterPlan, AttentionBlock, AttentionPlan, RotaryAxes  # noqa: E402


def grid(frames: int, height: int, width: int) -> torch.Tensor:
    """(t, h, w) of each token of a latent grid, time slowest."""
    return torch.cartesian_prod(torch.arange(frames), torch.arange(height), torch.arange(width)).int()


def main(requests=((9, 30, 54), (1, 30, 54), (5, 16, 24)), dim=5376, heads=8, head_dim=128, device=None) -> torch.Tensor:
    device = device or ("cuda" if torch.cuda.is_available() else "cpu")
    gen = torch.Generator().manual_seed(0)
    lengths = [t * h * w for t, h, w in requests]
    block = AttentionBlock(dim, heads, head_dim, 256, adapters=2, adapter_rank=32)
    for layer in (block.qkv, block.out):
        layer.qweight.copy_(torch.randint(-127, 128, layer.qweight.shape, generator=gen, dtype=torch.int8))
        layer.wscale.fill_(layer.in_features ** -0.5 / 73)
    for bank in (block.qkv_adapters, block.out_adapters):
        for i in range(bank.adapters):
            bank.load(i, torch.randn(32, bank.in_features, generator=gen) * bank.in_features ** -0.5,
                      torch.randn(bank.out_features, 32, generator=gen) * 32 ** -0.5, scale=0.5)
    block = block.to(device)

    plan = AttentionPlan(lengths, heads=heads, head_dim=head_dim, device=device)
    adapters = AdapterPlan([0, -1, 1], lengths, adapters=2, device=device)  # the second request takes none
    rotary = RotaryAxes((44, 42, 42), device=device)
    positions = torch.cat([grid(*r) for r in requests]).to(device)
    x = torch.randn(sum(lengths), dim, generator=gen).to(torch.bfloat16).to(device)
    y = block(x, plan, positions=positions, rotary=rotary, adapters=adapters)
    if y.is_cuda:
        torch.cuda.synchronize()
        began = time.perf_counter()
        for _ in range(10):
            y = block(x, plan, positions=positions, rotary=rotary, adapters=adapters)
        torch.cuda.synchronize()
        print(f"{sum(lengths)} tokens of {len(requests)} requests: {(time.perf_counter() - began) / 10 * 1e3:.3f} ms a block")
    return y


if __name__ == "__main__":
    print(main().shape)

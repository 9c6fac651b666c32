"""The attention block's operators as programs call them: from several threads, with copied plans, in place between other
layers, beyond 2^31 elements."""

from __future__ import annotations

import threading

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

"""The rotary calls captured once and replayed with other positions, slots and operands."""

from __future__ import annotations

import pytest
import torch

from kernelo_b200.kernels.rotary import rotary, rotary_table, rotary_to_cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_captured_in_a_graph(dtype, device):
    gen = torch.Generator(device=device).manual_seed(0)

    def fresh(*shape):
        return torch.randn(*shape, generator=gen, device=device).to(dtype)

    q, k, v = fresh(9, 8, 64), fresh(9, 2, 64), fresh(9, 2, 64)
    caches = [torch.zeros(5, 2, 16, 64, device=device, dtype=dtype) for _ in range(2)]
    table = rotary_table(500, 64, device=device)
    positions = torch.arange(9, dtype=torch.int32, device=device)
    slots = torch.arange(9, device=device)
    k_out = torch.empty_like(k)
    rotary_to_cache(q, k, v, positions, table, *caches, slots, k_out=k_out)  # the library is loaded
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        turned = rotary_to_cache(q, k, v, positions, table, *caches, slots, k_out=k_out)
        back = rotary(turned, k_out, positions, table, inverse=True)
    for seed in range(3):
        for t in (q, k, v):
            t.copy_(fresh(*t.shape))
        positions.copy_(torch.randint(0, 500, (9,), generator=gen, device=device, dtype=torch.int32))
        slots.copy_(torch.randperm(80, generator=gen, device=device)[:9])
        slots[seed] = -1
        want = [torch.zeros_like(c) for c in caches]
        want_k = torch.empty_like(k)
        want_q = rotary_to_cache(q, k, v, positions, table, *want, slots, k_out=want_k)
        want_back = rotary(want_q, want_k, positions, table, inverse=True)
        for c in caches:
            c.zero_()
        graph.replay()
        assert torch.equal(turned, want_q) and torch.equal(k_out, want_k)
        assert all(torch.equal(a, b) for a, b in zip((*caches, *back), (*want, *want_back)))

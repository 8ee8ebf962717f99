"""Workspaces of calls under capture: a graph's own, with counters that the graph clears."""

from __future__ import annotations

import pytest
import torch

from kernelo_b200.kernels.attention import tree_attention
from kernelo_b200.runtime import native

CPU = torch.device("cpu", 0)


@pytest.fixture
def pool(monkeypatch):
    """A pool on the host, and the capture that its next calls are in."""
    state = {"capture": 0}
    monkeypatch.setattr(native, "_capture_id", lambda stream: state["capture"], raising=False)
    return native._WorkspacePool(), state


def test_captures_get_workspaces_of_their_own(pool):
    pool, state = pool
    plain = pool.get(CPU, 7, 1 << 20)
    assert not plain.any() and pool.get(CPU, 7, 1 << 18) is plain
    kept = []
    for capture in (1, 2):
        state["capture"] = capture
        buf = pool.get(CPU, 7, 1 << 18)
        assert buf.data_ptr() not in [plain.data_ptr(), *(b.data_ptr() for b in kept)]
        assert not buf[:64 * 1024].any()
        buf[:8] = 1  # as a kernel of another graph, half-way
        assert pool.get(CPU, 7, 1 << 18) is buf, "calls of one capture share it"
        assert pool.get(CPU, 8, 1 << 18) is not buf, "but not on different streams"
        kept.append(buf)
    state["capture"] = 0
    assert pool.get(CPU, 7, 1 << 20) is plain


def test_the_first_call_of_a_stream_under_capture_leaves_nothing_to_later_ones(pool):
    """What clears a buffer under capture runs with the graph only."""
    pool, state = pool
    state["capture"] = 5
    buf = pool.get(CPU, 3, 1 << 18)
    state["capture"] = 6
    assert pool.get(CPU, 3, 1 << 18) is not buf
    state["capture"] = 0
    later = pool.get(CPU, 3, 1 << 18)
    assert later is not buf and not later.any()


def test_growth_outside_keeps_a_captured_workspace_and_the_other_way_round(pool):
    pool, state = pool
    plain = pool.get(CPU, 7, 1 << 18)
    state["capture"] = 9
    small = pool.get(CPU, 7, 1 << 18)
    large = pool.get(CPU, 7, 1 << 20)
    assert large.numel() >= 1 << 20 and large is not small and not large[:64 * 1024].any()
    state["capture"] = 0
    assert pool.get(CPU, 7, 1 << 18) is plain
    assert pool.get(CPU, 7, 1 << 21) is not large


def decode(device, context, seed):
    """One token each over a cache whose work is cut between CTAs."""
    gen = torch.Generator(device=device).manual_seed(seed)
    pages = [-(-(c + 1) // 16) for c in context]
    k, v = (torch.randn(sum(pages), 2, 16, 128, generator=gen, device=device).half() for _ in range(2))
    table = torch.full((len(context), max(pages)), -1, dtype=torch.int32, device=device)
    at = 0
    for r, n in enumerate(pages):
        table[r, :n] = torch.arange(at, at + n)
        at += n
    q = torch.randn(len(context), 8, 128, generator=gen, device=device).half()
    return q, k, v, table, torch.tensor(context, dtype=torch.int32, device=device)


@pytest.mark.gpu
def test_graphs_replayed_in_another_order_and_beside_one_another(device):
    native.workspaces.reset()
    calls = [decode(device, (3000, 50), 0), decode(device, (9000, 700, 20), 1)]
    graphs, outs = [], []
    for call in calls:  # nothing ran on the capturing stream before: no workspace of it exists
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append([tree_attention(*call) for _ in range(2)])
        graphs.append(graph)
    want = [tree_attention(*call) for call in calls]
    for g in (1, 0, 1):
        for out in outs[g]:
            out.zero_()
        graphs[g].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, want[g]) for out in outs[g])
    streams = [torch.cuda.Stream() for _ in graphs]
    for out in (*outs[0], *outs[1]):
        out.zero_()
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(out, want[g]) for g in range(2) for out in outs[g])
    # a larger call outside gets a larger workspace; the graphs' own stay
    large = decode(device, (500,) * 8, 2)
    masked = torch.cat([large[0]] * 8)
    tree_attention(masked, *large[1:], torch.arange(0, 65, 8, dtype=torch.int32, device=device))
    for g in (0, 1):
        graphs[g].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(out, want[g]) for g in range(2) for out in outs[g])
    assert native.device_status() == 0

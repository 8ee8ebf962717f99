"""A step that was planned, and what may happen to the cache before its tokens are the requests'."""

from __future__ import annotations

import pytest
import torch

from kernelo_b200.integration import PagedCache, ServingConfig, serving
from kernelo_b200.integration.serving import Step

SMALL = ServingConfig(hidden=64, heads=2, kv_heads=2, intermediate=64, block_size=4, max_positions=64)


def planned(lens, new_lens):
    """A cache on the host and a step, as `plan` leaves them: pages in order, those of the step still in the free list."""
    cache = PagedCache(SMALL, requests=len(lens), blocks=20, dtype=torch.float32, device="cpu")
    cache.lens, at = list(lens), 0
    for r, n in enumerate(lens):
        pages = -(-n // 4)
        cache.block_table[r, :pages] = torch.arange(at, at + pages, dtype=torch.int32)
        at += pages
    cache.free, taken = cache.free[at:], at
    for r, (n, a) in enumerate(zip(lens, new_lens)):
        pages = range(-(-n // 4), -(-(n + a) // 4))
        cache.block_table[r, pages.start:pages.stop] = torch.arange(taken, taken + len(pages), dtype=torch.int32)
        taken += len(pages)
    return cache, Step(tuple(new_lens), None, None, tuple(lens), cache._moved)


@pytest.mark.parametrize("lens,new,parents,children", [
    ((6, 0, 0), (1, 0, 5), [0], [1]),  # the fork takes the page that the step's prompt has
    ((6, 0, 0), (1, 0, 5), [0], [2]),  # the step's row becomes another request's
    ((0, 0, 0), (5, 0, 0), [1], [0]),  # of nothing: the row with the step's pages is cleared, and all lengths stay
    ((8, 0, 0), (1, 0, 0), [0], [1]),
])
def test_a_step_planned_before_a_fork_is_refused(lens, new, parents, children, monkeypatch):
    monkeypatch.setattr(serving, "fork_requests", lambda *args: None)
    cache, step = planned(lens, new)
    cache.check_step(step)
    cache.fork([], [])  # of nobody
    cache.check_step(step)
    cache.fork(parents, children)
    held = list(cache.lens), cache.free.tolist()
    with pytest.raises(ValueError, match="planned before"):
        cache.check_step(step)
    with pytest.raises(ValueError, match="planned before"):
        cache.advance(step)
    assert held == (list(cache.lens), cache.free.tolist())


def test_a_fork_that_is_refused_leaves_a_step_as_it_was():
    cache, step = planned((6, 3, 0), (1, 1, 0))
    with pytest.raises(ValueError, match="have tokens"):
        cache.fork([0], [1])
    cache.advance(step)
    assert cache.lens == [7, 4, 0]


@pytest.mark.parametrize("released", [1, [1], [1, 2], []])
def test_a_release_of_requests_without_tokens_leaves_a_step_as_it_was(released):
    cache, step = planned((6, 0, 0), (3, 5, 0))
    table, free = cache.block_table.clone(), cache.free.tolist()
    cache.release(released)
    assert torch.equal(cache.block_table, table) and cache.free.tolist() == free
    cache.advance(step)
    assert cache.lens == [9, 5, 0] and cache.free.tolist() == list(range(5, 20))
    assert cache.block_table[0, :3].tolist() == [0, 1, 2] and cache.block_table[1, :2].tolist() == [3, 4]


@pytest.mark.gpu
def test_requests_without_tokens_released_and_forked_beside_a_step(device):
    cache = PagedCache(SMALL, requests=4, blocks=20, device=device)
    cache.advance(cache.plan([6, 0, 0, 0]))
    step = cache.plan([1, 5, 0, 0])
    cache.release([1, 2])
    cache.advance(step)
    held = [cache.block_table[r, :2].tolist() for r in range(2)]
    assert cache.lens == [7, 5, 0, 0] and sorted([*held[0], *held[1], *cache.free.tolist()]) == list(range(20))
    step = cache.plan([1, 1, 3, 0])
    cache.fork([0], [3])
    with pytest.raises(ValueError, match="planned before"):
        cache.advance(step)
    cache.advance(cache.plan([1, 1, 3, 1]))
    assert cache.lens == [8, 6, 3, 8]
    held = [p for r in range(4) for p in cache.block_table[r, :-(-cache.lens[r] // 4)].tolist()]
    assert len(held) == 2 + 2 + 1 + 2 and held.count(held[0]) == 2
    assert sorted([*set(held), *cache.free.tolist()]) == list(range(20))

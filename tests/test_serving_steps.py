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

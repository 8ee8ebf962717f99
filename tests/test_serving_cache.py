"""What a paged cache keeps of a step's tokens, and what it gives back."""

from __future__ import annotations

import pytest
import torch

from kernelo_b200.integration import PagedCache, ServingConfig
from kernelo_b200.integration.serving import Step
from kernelo_b200.testing import assert_verified
from tests.test_serving import TINY, make_block, plain_block

SMALL = ServingConfig(hidden=64, heads=2, kv_heads=2, intermediate=64, block_size=4, max_positions=64)


def planned(lens, new_lens):
    """A cache on the host as `plan` leaves it for requests of those lengths: keys and values say request and place."""
    cache = PagedCache(SMALL, requests=len(lens), blocks=40, dtype=torch.float32, device="cpu")
    order = torch.randperm(40, generator=torch.Generator().manual_seed(0)).int()
    cache.k.zero_()
    cache.lens, at = list(lens), 0
    for r, (n, a) in enumerate(zip(lens, new_lens)):
        for col in range(-(-(n + a) // 4)):
            cache.block_table[r, col] = order[at]
            at += 1
        for place in range(n + a):
            page = cache.block_table[r, place // 4].long()
            cache.k[page, :, place % 4] = 1000 * r + place
            cache.v[page, :, place % 4] = -1000 * r - place
    held = sum(-(-n // 4) for n in lens)
    # the pages that the step took come first in the free list; which ones they are does not matter here
    cache.free = torch.cat([torch.zeros(at - held, dtype=torch.int32), order[at:]])
    return cache, Step(tuple(new_lens), None, None)


def held(cache, r):
    """The keys of request r, place by place."""
    at = torch.arange(cache.lens[r])
    page = cache.block_table[r].long()[at // 4]
    assert torch.equal(cache.k[page, 0, at % 4], -cache.v[page, 1, at % 4])
    return [int(x) for x in cache.k[page, 1, at % 4, 0]]


@pytest.mark.parametrize("paths", [([0, 1, 3], [0], [], 2), ([1], [4, 5, 6], [2, 3], 0), ([0, 1, 2, 3, 4], [6], [0, 2], [0, 1, 2])])
def test_an_accepted_branch_is_moved_together(paths):
    lens, new = (5, 8, 0, 3), (5, 7, 4, 3)
    cache, step = planned(lens, new)
    cache.advance(step, kept=paths)
    for r, path in enumerate(paths):
        path = range(path) if isinstance(path, int) else path
        want = [*range(lens[r]), *(lens[r] + i for i in path)]
        assert held(cache, r) == [1000 * r + i for i in want]
    assert cache.free.shape[0] == 40 - sum(-(-n // 4) for n in cache.lens)


@pytest.mark.parametrize("kept", [[[1, 0], 1], [[0, 0], 1], [[-1], 1], [[0, 5], 1], [6, 0], [-1, 0], [range(-1, 1), 0], [[0]], [[0], 1, 1]])
def test_what_is_no_branch_is_refused(kept):
    cache, step = planned((5, 8), (5, 7))
    before = cache.k.clone()
    with pytest.raises(ValueError, match="kept"):
        cache.advance(step, kept=kept)
    assert cache.lens == [5, 8] and torch.equal(cache.k, before)


def test_a_released_request_gives_its_pages_back():
    cache, step = planned((5, 8, 0), (4, 0, 3))
    cache.advance(step)
    taken = [cache.block_table[r, :-(-n // 4)].tolist() for r, n in enumerate(cache.lens)]
    free = cache.free.tolist()
    cache.release(1)
    cache.release(2)
    assert cache.lens == [9, 0, 0] and cache.free.tolist() == free + taken[1] + taken[2]
    assert cache.block_table[0, :3].tolist() == taken[0] and (cache.block_table[1:] == -1).all()
    cache.release(1)  # of nothing
    assert cache.free.shape[0] == 37
    for request in (3, -1):
        with pytest.raises(ValueError, match="request must be"):
            cache.release(request)


def test_a_step_planned_for_other_lengths_is_refused():
    cache, step = planned((5, 8), (1, 1))
    step = Step(step.new_lens, None, None, (5, 8))
    cache.advance(step)
    with pytest.raises(ValueError, match="planned"):
        cache.advance(step)
    cache, _ = planned((5, 8), (1, 1))
    cache.release(0)
    with pytest.raises(ValueError, match="planned"):
        cache.advance(step)


@pytest.mark.gpu
def test_a_server_goes_on_with_the_pages_of_finished_requests(device):
    """More requests one after another than the cache has pages for at once."""
    block = make_block(torch.float16, device)
    cache = PagedCache(TINY, requests=2, blocks=6, device=device)  # 48 tokens
    gen = torch.Generator(device=device).manual_seed(3)
    with torch.inference_mode():
        for turn in range(5):
            row = turn % 2
            lens = [0, 0]
            lens[row] = 17 + turn
            x, step = torch.randn(17 + turn, TINY.hidden, generator=gen, device=device).half(), cache.plan(lens)
            got = block.prompts(x, cache, step)
            at = torch.arange(17 + turn, device=device)
            want = plain_block(block, x, at, at[None, :] <= at[:, None])
            assert_verified(want, got, dtype=torch.float16, context="prompt")
            cache.advance(step)
            y, step = torch.randn(1, TINY.hidden, generator=gen, device=device).half(), cache.plan([int(r == row) for r in range(2)])
            got = block.tokens(y, cache, step)
            at = torch.arange(18 + turn, device=device)
            want = plain_block(block, torch.cat([x, y]), at, at[None, :] <= at[:, None])[-1:]
            assert_verified(want, got, dtype=torch.float16, context="token")
            cache.advance(step)
            cache.release(row)
        assert sorted(cache.free.tolist()) == list(range(6))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_tokens_after_an_accepted_branch(dtype, device):
    """Nodes 1 and 2 follow 0, node 3 follows 1: 0-1-3 or 0-2 are kept, and ordinary tokens follow."""
    block = make_block(dtype, device)
    cache = PagedCache(TINY, requests=2, blocks=40, dtype=dtype, device=device)
    gen = torch.Generator(device=device).manual_seed(1)

    def fresh(lens):
        return [torch.randn(n, TINY.hidden, generator=gen, device=device).to(dtype) for n in lens]

    with torch.inference_mode():
        history, step = fresh((13, 30)), cache.plan((13, 30))
        block.prompts(torch.cat(history), cache, step)
        cache.advance(step)
        parts, step = fresh((4, 4)), cache.plan((4, 4))
        words = torch.tensor([[0b0001], [0b0011], [0b0101], [0b1011]] * 2, device=device)
        block.tokens(torch.cat(parts), cache, step, words, torch.tensor([0, 1, 1, 2] * 2, dtype=torch.int32, device=device))
        branches = ([0, 1, 3], [0, 2])
        cache.advance(step, kept=branches)
        assert cache.lens == [16, 32]
        history = [torch.cat([h, x[b]]) for h, x, b in zip(history, parts, branches)]
        parts, step = fresh((1, 3)), cache.plan((1, 3))
        got = block.tokens(torch.cat(parts), cache, step)
        want = []
        for h, x in zip(history, parts):
            n = h.shape[0] + x.shape[0]
            at = torch.arange(n, device=device)
            want.append(plain_block(block, torch.cat([h, x]), at, at[None, :] <= at[:, None])[h.shape[0]:])
        assert_verified(torch.cat(want), got, dtype=dtype, context="tokens after a branch")

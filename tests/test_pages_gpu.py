"""Pages when requests fork, end and are moved together, against the definition page by page. Everything is a whole number
or a copy: results are equal."""

from __future__ import annotations

import random

import pytest
import torch

from kernelo_b200.kernels.paged import build_slots, compact_pages, fork_requests, release_requests

pytestmark = pytest.mark.gpu


class Pool:
    """Caches, a table, lengths, holders and free pages on the GPU, and the same as Python numbers."""

    def __init__(self, lens, device, *, blocks=60, block=16, cols=12, heads=2, dim=32, caches=2, dtype=torch.bfloat16,
                 share=(), seed=0, make=None):
        rng = random.Random(seed)
        order = list(range(blocks))
        rng.shuffle(order)
        self.block, self.lens = block, list(lens)
        self.table = [[-1] * cols for _ in lens]
        for r, n in enumerate(lens):
            for col in range(-(-n // block)):
                self.table[r][col] = order.pop()
        for a, b, n in share:  # request b's first n pages are those of a
            for col in range(n):
                order.append(self.table[b][col])
                self.table[b][col] = self.table[a][col]
        self.free = order
        count = [0] * blocks
        for r, n in enumerate(lens):
            for col in range(-(-n // block)):
                count[self.table[r][col]] += 1
        self.holders = [max(c - 1, 0) for c in count]
        gen = torch.Generator().manual_seed(seed)
        make = make or (lambda c: torch.randn(blocks, heads, block, dim, generator=gen).to(dtype).to(device))
        self.caches = [make(c) for c in range(caches)]
        self.device = device
        self.upload()

    def ints(self, values):
        return torch.tensor(values, dtype=torch.int32, device=self.device)

    def upload(self):
        self.d_table, self.d_lens, self.d_holders, self.d_free = map(self.ints, (self.table, self.lens, self.holders, self.free))
        self.want = [c.clone() for c in self.caches]

    def check(self):
        assert self.d_table.tolist() == self.table
        assert self.d_lens.tolist() == self.lens
        assert self.d_holders.tolist() == self.holders
        for got, want in zip(self.caches, self.want):
            assert torch.equal(got, want)

    def fork(self, parents, children):
        got = fork_requests(self.caches, self.d_table, self.d_lens, self.d_holders, self.d_free, self.ints(parents),
                            self.ints(children))
        taken = dropped = 0
        rows = len(self.table)
        for p, c in zip(parents, children):
            if not (0 <= p < rows and 0 <= c < rows) or children.count(c) > 1 or c in parents:
                dropped += 1
                continue
            n = min(max(self.lens[p], 0), len(self.table[p]) * self.block)
            full, tail = divmod(n, self.block)
            self.table[c] = [self.table[p][col] if col < full else -1 for col in range(len(self.table[c]))]
            for page in self.table[c][:full]:
                if 0 <= page < len(self.holders):
                    self.holders[page] += 1
            self.lens[c] = n
            if tail:
                if taken < len(self.free):
                    page, source = self.free[taken], self.table[p][full]
                    self.table[c][full] = page
                    if 0 <= source < len(self.holders):
                        for want in self.want:
                            want[page, :, :tail] = want[source, :, :tail]
                else:
                    dropped += 1
                taken += 1
        assert got.blocks_taken.tolist() == [taken] and got.dropped.tolist() == [dropped]
        self.free = self.free[taken:]
        self.d_free = self.ints(self.free)

    def release(self, requests):
        got = release_requests(self.d_table, self.d_lens, self.d_holders, self.ints(requests), block_size=self.block)
        rows, cols = len(self.table), len(self.table[0])
        done, entries = set(), []
        for r in requests:
            if 0 <= r < rows and r not in done:
                done.add(r)
                held = min(-(-max(self.lens[r], 0) // self.block), cols)
                entries += [p for p in self.table[r][:held] if 0 <= p < len(self.holders)]
                self.table[r], self.lens[r] = [-1] * cols, 0
        for p in entries:
            self.holders[p] -= 1
        freed = list(dict.fromkeys(p for p in entries if self.holders[p] < 0))
        for p in freed:
            self.holders[p] = 0
        assert got.count.tolist() == [len(freed)]
        assert got.pages.tolist() == freed + [-1] * (len(requests) * cols - len(freed))
        self.free = self.free + freed
        self.d_free = self.ints(self.free)

    def compact(self):
        got = compact_pages(self.caches, self.d_table, self.d_lens, self.d_holders)
        blocks, cols = len(self.holders), len(self.table[0])
        held = [min(-(-max(n, 0) // self.block), cols) for n in self.lens]
        live = sorted({p for row, n in zip(self.table, held) for p in row[:n] if 0 <= p < blocks})
        count = len(live)
        holes = sorted(set(range(count)) - set(live))
        moves = dict(zip([p for p in live if p >= count], holes))
        renamed = [-1] * blocks
        for p in live:
            renamed[p] = moves.get(p, p)
        for want in self.want:
            want[list(moves.values())] = want[list(moves)]
        self.table = [[renamed[p] if col < n and 0 <= p < blocks else p for col, p in enumerate(row)]
                      for row, n in zip(self.table, held)]
        holders = [0] * blocks
        for p in live:
            holders[renamed[p]] = self.holders[p]
        self.holders, self.free = holders, list(range(count, blocks))
        assert got.live.tolist() == [count] and got.moves.tolist() == [len(moves)]
        assert got.renamed.tolist() == renamed
        self.d_free = self.ints(self.free)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("block,dim,heads,caches", [(16, 32, 2, 2), (8, 128, 8, 1), (5, 7, 3, 3), (1, 64, 1, 2), (64, 20, 1, 2),
                                                    (16, 1, 2, 2)])
def test_fork_of_every_tail(block, dim, heads, caches, dtype, device):
    """Parents with no token, a page less one, a page and one more: each answered twice."""
    lens = [0, 1, block - 1, block, block + 1, 3 * block - 1 if block > 1 else 2] + [0] * 13
    pool = Pool(lens, device, block=block, dim=dim, heads=heads, caches=caches, dtype=dtype)
    children = list(range(6, 18))
    random.Random(0).shuffle(children)
    pool.fork([0, 1, 2, 3, 4, 5] * 2, children)
    pool.check()


def test_one_parent_many_children_and_forks_of_forks(device):
    pool = Pool([40, 33] + [0] * 10, device)
    pool.fork([0] * 4 + [1] * 2, [2, 3, 4, 5, 6, 7])
    pool.check()
    pool.fork([3, 7, 0], [8, 9, 10])
    pool.check()
    pool.release([0, 3])
    pool.check()
    pool.release([8, 2, 4, 5, 10])
    pool.check()
    pool.compact()
    pool.check()
    pool.release([1, 6, 7, 9, 11])
    pool.check()
    assert sorted(pool.free) == list(range(60)) and pool.holders == [0] * 60


def test_pairs_that_do_nothing(device):
    pool = Pool([40, 20, 30] + [0] * 8, device)
    # a child that is a parent, one named twice, rows that are none, a request of itself; good ones among them
    pool.fork([0, 1, 2, 0, 1, -1, 2 ** 31 - 1, 0, 1, 2, 11], [1, 3, 3, 11, -1, 4, 5, 6, 7, 2, 8])
    pool.check()
    pool.fork([], [])
    pool.check()


def test_a_free_list_that_ends(device):
    pool = Pool([40, 20, 16] + [0] * 8, device, blocks=9)
    assert len(pool.free) == 3
    pool.fork([0, 2, 1, 0, 1, 0], [3, 4, 5, 6, 7, 8])
    pool.check()
    assert pool.table[7] != [-1] * 12 and pool.table[7][1] == -1


@pytest.mark.parametrize("caches", [64, 65, 130])
def test_many_caches(caches, device):
    pool = Pool([20, 37, 0, 0], device, caches=caches, blocks=14, dim=8)
    pool.fork([0, 1], [2, 3])
    pool.check()
    pool.release([1])
    pool.compact()
    pool.check()


def test_numbers_that_are_no_pages(device):
    """Entries outside the pool are carried, never followed."""
    pool = Pool([40, 20, 50, 0, 0, 0], device)
    pool.table[0][1], pool.table[1][1], pool.table[2][0] = 60, -1, 2 ** 31 - 1
    pool.lens[2] = 12 * 16 + 5  # more tokens than a row has pages for
    pool.upload()
    pool.fork([0, 1, 2], [3, 4, 5])
    pool.check()
    pool.lens[5] = -3
    pool.upload()
    pool.release([3, 1, 5])
    pool.check()
    pool.compact()
    pool.check()


def orders(device, dtype=torch.bfloat16):
    def slots_first(c):
        return torch.randn(60, 16, 2, 32, device=device).to(dtype).transpose(1, 2)

    def apart(c):
        return torch.randn(120, 3, 19, 40, device=device).to(dtype)[::2, 1:, 2:18, 8:]

    def odd(c):
        return torch.randn(60, 2, 16, 35, device=device).to(dtype)[..., 2 + c:34 + c]

    def half(c):
        return torch.randn(60, 4, 16, 32, device=device).to(dtype)[:, 2 * (c % 2):2 + 2 * (c % 2)]

    return {"slots_first": slots_first, "apart": apart, "odd": odd, "half": half}


@pytest.mark.parametrize("order", ["slots_first", "apart", "odd", "half"])
def test_caches_of_other_orders(order, device):
    torch.manual_seed(0)
    pool = Pool([40, 33, 100] + [0] * 4, device, make=orders(device)[order])
    pool.fork([0, 1, 2, 2], [3, 4, 5, 6])
    pool.check()
    pool.release([2, 0])
    pool.compact()
    pool.check()


def test_a_table_in_a_wider_buffer(device):
    pool = Pool([40, 33] + [0] * 4, device)
    wide = torch.full((6, 20), 99, dtype=torch.int32, device=device)
    wide[:, 3:15] = pool.d_table
    pool.d_table = wide[:, 3:15]
    pool.fork([0, 1, 0], [2, 3, 4])
    pool.release([0, 0, 7, -1])
    pool.compact()
    pool.check()
    assert (wide[:, :3] == 99).all() and (wide[:, 15:] == 99).all()


@pytest.mark.parametrize("requests,longest,blocks", [(3, 100, 60), (40, 900, 2400), (200, 700, 9000), (300, 2000, 40000)])
def test_release_and_compact_of_many(requests, longest, blocks, device):
    """Requests that share pages in groups, released a part at a time in any order, some named twice."""
    rng = random.Random(requests)
    lens = [rng.randint(0, longest) for _ in range(requests)]
    share = [(r // 5 * 5, r, rng.randint(0, min(lens[r], lens[r // 5 * 5]) // 16)) for r in range(requests) if r % 5]
    pool = Pool(lens, device, blocks=blocks, cols=longest // 16 + 2, heads=1, dim=2, share=share)
    left = list(range(requests))
    rng.shuffle(left)
    while left:
        n = rng.randint(1, requests // 2 + 1)
        now, left = left[:n], left[n:]
        pool.release(now + now[:2])
        pool.check()
        pool.compact()
        pool.check()
    assert sorted(pool.free) == list(range(blocks))


@pytest.mark.parametrize("blocks", [1, 31, 32, 33, 64, 8192, 8193, 70000])
def test_compact_at_the_edges(blocks, device):
    """An empty pool, a full one, all live pages first, all of them last."""
    def make(c):
        return torch.randn(blocks, 1, 1, 2, device=device).half()

    for held in ([], range(blocks), range(blocks // 2), range(blocks - blocks // 3, blocks), range(0, blocks, 2)):
        pool = Pool([0] * 2, device, blocks=blocks, block=1, cols=blocks, make=make)
        held = list(held)
        random.Random(1).shuffle(held)
        pool.table[1][:len(held)], pool.lens[1] = held, len(held)
        pool.upload()
        pool.compact()
        pool.check()


def test_an_empty_table_and_no_requests(device):
    pool = Pool([20, 30], device)
    pool.release([])
    pool.check()
    empty = torch.empty(0, 12, dtype=torch.int32, device=device)
    none = torch.empty(0, dtype=torch.int32, device=device)
    assert compact_pages(pool.caches, empty, none, pool.d_holders).live.tolist() == [0]
    assert compact_pages(pool.caches, empty.view(0, 12)[:, :0], none, pool.d_holders).live.tolist() == [0]
    thin = torch.empty(2, 0, dtype=torch.int32, device=device)
    assert compact_pages(pool.caches, thin, pool.d_lens, pool.d_holders).live.tolist() == [0]
    assert release_requests(thin, pool.d_lens.clone(), pool.d_holders, none, block_size=16).count.tolist() == [0]


def test_pages_beyond_32_bit_offsets(device):
    """Pages that begin beyond 2^31 elements and 2^32 bytes."""
    blocks, pages = 40, 1 << 27
    big = torch.zeros(blocks * pages // 2, dtype=torch.float16, device=device)  # 5 GB
    cache = big.view(blocks, 1, 16, pages // 32)[..., :64]
    table = torch.full((3, 4), -1, dtype=torch.int32, device=device)
    table[0, :2] = torch.tensor([39, 38], dtype=torch.int32)
    lens = torch.tensor([20, 0, 0], dtype=torch.int32, device=device)
    holders = torch.zeros(blocks, dtype=torch.int32, device=device)
    cache[38] = torch.randn(1, 16, 64, device=device).half()
    cache[39] = torch.randn(1, 16, 64, device=device).half()
    ints = dict(dtype=torch.int32, device=device)
    fork_requests([cache], table, lens, holders, torch.tensor([37], **ints), torch.tensor([0], **ints), torch.tensor([1], **ints))
    assert table[1].tolist() == [39, 37, -1, -1]
    assert torch.equal(cache[37, :, :4], cache[38, :, :4]) and not cache[37, :, 4:].any()
    before = [cache[p].clone() for p in (37, 38, 39)]
    got = compact_pages([cache], table, lens, holders)
    assert got.live.tolist() == [3] and all(torch.equal(cache[p], b) for p, b in enumerate(before))
    assert table[:2, :2].tolist() == [[2, 1], [2, 0]] and holders[:3].tolist() == [0, 0, 1]


def test_captured_and_replayed_with_other_requests(device):
    """A step that forks, plans the children's next tokens, and ends requests, captured once."""
    pool = Pool([40, 33] + [0] * 6, device, blocks=60)
    parents, children, ended = pool.ints([0, 0]), pool.ints([2, 3]), pool.ints([0])
    added, state = pool.ints([0, 1, 1, 1, 0, 0, 0, 0]), (pool.d_table, pool.d_lens, pool.d_holders, *pool.caches)
    start = [x.clone() for x in state]

    def step():
        forked = fork_requests(pool.caches, pool.d_table, pool.d_lens, pool.d_holders, pool.d_free, parents, children)
        slots = build_slots(pool.d_lens, added, pool.d_table, pool.d_free[8:], block_size=16, max_tokens=4)
        freed = release_requests(pool.d_table, pool.d_lens, pool.d_holders, ended, block_size=16)
        packed = compact_pages(pool.caches, pool.d_table, pool.d_lens, pool.d_holders)
        return [*forked, *slots, *freed, packed.renamed, packed.live]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for lists in (([0, 0], [2, 3], [0]), ([1, 0], [4, 5], [1]), ([1, 1], [7, 3], [7])):
        for to, values in zip((parents, children, ended), lists):
            to.copy_(pool.ints(values))
        for to, x in zip(state, start):
            to.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        seen = [x.clone() for x in (*captured, *state)]
        for to, x in zip(state, start):
            to.copy_(x)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            eager = step()
        side.synchronize()
        for a, b in zip(seen, (*eager, *state)):
            assert torch.equal(a, b)


def test_many_released_captured_and_replayed(device):
    """Enough entries for a launch of each phase: a graph of them, replayed beside eager calls on another stream."""
    rng = random.Random(3)
    lens = [rng.randint(0, 2000) for _ in range(300)]
    share = [(r // 5 * 5, r, rng.randint(0, min(lens[r], lens[r // 5 * 5]) // 16)) for r in range(300) if r % 5]
    pool = Pool(lens, device, blocks=40000, cols=130, heads=1, dim=2, caches=1, share=share)
    ended = pool.ints(rng.sample(range(300), 290))
    state = (pool.d_table, pool.d_lens, pool.d_holders)
    start = [x.clone() for x in state]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        release_requests(*state, ended, block_size=16)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = release_requests(*state, ended, block_size=16)
    for seed in range(3):
        ended.copy_(pool.ints(random.Random(seed).sample(range(300), 290)))
        for to, x in zip(state, start):
            to.copy_(x)
        graph.replay()
        graph.replay()  # of requests that have ended: nothing
        assert captured.count.item() == 0
        for to, x in zip(state, start):
            to.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        seen = [x.clone() for x in (*captured, *state)]
        for to, x in zip(state, start):
            to.copy_(x)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            eager = release_requests(*state, ended, block_size=16)
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(seen, (*eager, *state)))
    for to, x in zip(state, start):
        to.copy_(x)
    pool.release(ended.tolist())
    pool.check()


def test_refusals(device):
    pool = Pool([40, 33, 0, 0], device)
    table, lens, holders, free = pool.d_table, pool.d_lens, pool.d_holders, pool.d_free
    one = pool.ints([0])
    good = dict(caches=pool.caches, block_table=table, context_lens=lens, holders=holders)
    other = pool.caches[0].transpose(1, 2).contiguous().transpose(1, 2)
    for change, message in ((dict(caches=[]), "at least one"), (dict(caches=[pool.caches[0], pool.caches[1].float()]), "one type"),
                            (dict(caches=[pool.caches[0], other]), "strides"),
                            (dict(caches=[c[:30] for c in pool.caches]), "holders must have shape"),
                            (dict(caches=[pool.caches[0][0]]), "expected caches"),
                            (dict(caches=[c.cpu() for c in pool.caches]), "caches must be on"),
                            (dict(caches=[pool.caches[0][:1].expand(60, -1, -1, -1)]), "overlap themselves"),
                            (dict(caches=[c.transpose(2, 3) for c in pool.caches]), "contiguous last"),
                            (dict(block_table=table.long()), "block_table must be int32"),
                            (dict(block_table=table.t()), "contiguous rows"),
                            (dict(block_table=table[:1].expand(4, -1)), "contiguous rows"),
                            (dict(block_table=table.cpu()), "CUDA tensor"),
                            (dict(context_lens=lens[:2]), "context_lens must have shape"),
                            (dict(holders=holders.long()), "holders must be"), (dict(holders=holders[:30]), "holders must have shape")):
        with pytest.raises(ValueError, match=message):
            compact_pages(**(good | change))
        with pytest.raises(ValueError, match=message):
            fork_requests(**(good | change), free_blocks=free, parents=one, children=one)
    for change, message in ((dict(parents=one.long()), "parents must be"), (dict(children=pool.ints([2, 3])), "one shape"),
                            (dict(free_blocks=free[None]), "one dimension"), (dict(children=one.cpu()), "children must be on")):
        with pytest.raises(ValueError, match=message):
            fork_requests(**(good | dict(free_blocks=free, parents=one, children=one) | change))
    for requests, size, message in ((one.long(), 16, "requests must be"), (one, 0, "block_size"), (one[None], 16, "one dimension")):
        with pytest.raises(ValueError, match=message):
            release_requests(table, lens, holders, requests, block_size=size)
    pool.check()

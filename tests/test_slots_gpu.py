"""Block tables and slot maps built from request lengths, against a loop on the host (whole numbers: equal)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from kernelo_b200.kernels.paged import build_slots

pytestmark = pytest.mark.gpu


def plan(context, new, table, free, block, most):
    """The definition, token by token."""
    table, taken, dropped, total = table.copy(), 0, 0, 0
    cu, positions, slots = [0], [0] * most, [-1] * most
    for r, (c, n) in enumerate(zip(context, new)):
        for col in range(-(-c // block), -(-(c + n) // block)):
            if col < table.shape[1]:
                table[r, col] = free[taken] if taken < len(free) else -1
            taken += 1
        for i in range(n):
            pos = c + i
            col = pos // block
            page = table[r, col] if col < table.shape[1] else -1
            slot = int(page) * block + pos % block if page >= 0 else -1
            if total < most:
                positions[total], slots[total] = pos, slot
            dropped += total >= most or slot < 0
            total += 1
        cu.append(total)
    return cu, positions, slots, taken, dropped, table


def check(context, new, block, device, *, columns=None, free=None, most=None, seed=0):
    rng = np.random.default_rng(seed)
    context, new = list(map(int, context)), list(map(int, new))
    held = [-(-c // block) for c in context]
    after = [-(-(c + n) // block) for c, n in zip(context, new)]
    columns = max([*after, 1]) + 2 if columns is None else columns
    total = sum(after) + 4
    order = rng.permutation(total).astype(np.int32)
    table = np.full((len(context), columns), -1, dtype=np.int32)
    at = 0
    for r, n in enumerate(held):
        table[r, :min(n, columns)] = order[at:at + n][:columns]
        at += n
    pool = order[at:] if free is None else order[at:at + free]
    most = sum(new) + 3 if most is None else most
    want = plan(context, new, table, pool, block, most)
    def to(a):
        return torch.tensor(np.asarray(a), dtype=torch.int32, device=device)

    wide = torch.full((len(context), columns + 3), -7, dtype=torch.int32, device=device)
    wide[:, 1:1 + columns] = torch.from_numpy(table).to(device)
    view = wide[:, 1:1 + columns]
    for _ in range(2):  # the same lengths again write the same values
        got = build_slots(to(context), to(new), view, to(pool), block_size=block, max_tokens=most)
        assert got.cu_new.tolist() == want[0]
        assert got.positions.tolist() == want[1]
        assert got.slots.tolist() == want[2]
        assert got.blocks_taken.tolist() == [want[3]]
        assert got.dropped.tolist() == [want[4]]
        assert np.array_equal(view.cpu().numpy(), want[5])
        assert (wide[:, 0] == -7).all() and (wide[:, columns + 1:] == -7).all()
    return got


@pytest.mark.parametrize("block", [1, 3, 16, 64])
def test_ragged_batches(block, device):
    rng = np.random.default_rng(block)
    for seqs, most_context, most_new in ((1, 0, 1), (1, 100, 1), (2, 5, 300), (64, 400, 1), (300, 40, 20), (700, 90, 5),
                                         (1537, 9, 3)):
        check(rng.integers(0, most_context + 1, seqs), rng.integers(0, most_new + 1, seqs), block, device)


def test_lengths_of_zero_and_whole_pages(device):
    check([0, 16, 15, 32, 0, 17], [0, 0, 1, 16, 16, 15], 16, device)
    check([0] * 5, [0] * 5, 16, device)
    check([], [], 16, device)
    check([5], [0], 16, device, most=0)


def test_one_long_prompt(device):
    check([7], [70001], 16, device)


def test_free_list_runs_out(device):
    for free in (0, 1, 3, 6):
        check([10, 0, 33, 16], [30, 20, 1, 40], 16, device, free=free)


def test_rows_and_outputs_too_short(device):
    check([10, 0, 33], [30, 80, 40], 16, device, columns=3)
    check([10, 0, 33], [30, 80, 40], 16, device, columns=1)
    check([10, 0, 33], [30, 80, 40], 16, device, most=50)
    check([10, 0, 33], [30, 80, 40], 16, device, most=0)


def test_held_pages_that_are_missing_give_no_slot(device):
    table = torch.tensor([[4, -1, -1]], dtype=torch.int32, device=device)
    got = build_slots(torch.tensor([20], dtype=torch.int32, device=device),
                      torch.tensor([14], dtype=torch.int32, device=device), table,
                      torch.tensor([9], dtype=torch.int32, device=device), block_size=16, max_tokens=14)
    assert got.slots.tolist() == [-1] * 12 + [144, 145] and got.dropped.tolist() == [12]


def test_captured_in_a_graph(device):
    context = torch.tensor([3, 30], dtype=torch.int32, device=device)
    new = torch.tensor([1, 1], dtype=torch.int32, device=device)
    table = torch.tensor([[0, -1, -1], [1, 2, -1]], dtype=torch.int32, device=device)
    free = torch.tensor([7, 8, 9], dtype=torch.int32, device=device)
    build_slots(context, new, table, free, block_size=16, max_tokens=4)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = build_slots(context, new, table, free, block_size=16, max_tokens=4)
    graph.replay()
    assert got.slots.tolist() == [3, 46, -1, -1]
    context.copy_(torch.tensor([16, 31], dtype=torch.int32))
    new.copy_(torch.tensor([1, 2], dtype=torch.int32))
    graph.replay()
    assert got.slots.tolist() == [112, 47, 128, -1] and table.tolist() == [[0, 7, -1], [1, 2, 8]]


def test_refusals(device):
    lens = torch.tensor([3, 30], dtype=torch.int32, device=device)
    table = torch.zeros(2, 3, dtype=torch.int32, device=device)
    free = torch.arange(4, dtype=torch.int32, device=device)
    good = dict(context_lens=lens, new_lens=lens, block_table=table, free_blocks=free, block_size=16, max_tokens=40)
    bad = [
        (dict(block_size=0), "block_size"), (dict(max_tokens=-1), "max_tokens"), (dict(block_table=table[0]), "int32"),
        (dict(block_table=table.long()), "block_table must be int32"), (dict(block_table=table.cpu()), "CUDA"),
        (dict(block_table=table.t()), "contiguous rows"), (dict(context_lens=lens[:1]), "context_lens must have"),
        (dict(new_lens=lens.long()), "new_lens must be"), (dict(new_lens=lens.cpu()), "new_lens must be on"),
        (dict(free_blocks=free[None]), "free_blocks"), (dict(free_blocks=free.long()), "free_blocks must be"),
    ]
    for change, message in bad:
        with pytest.raises(ValueError, match=message):
            build_slots(**(good | change))

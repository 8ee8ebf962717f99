"""Pages of a key/value cache, and the plan of a serving step built on the GPU.

:func:`build_slots` takes the lengths of a batch's requests and writes, in one
launch, everything that the step's other calls read: new pages into the block
table, and the offset, position and cache slot of every added token. Nothing is
read on the host, so it can be captured with the step.

Requests may hold pages together: :func:`fork_requests` answers one prompt several
ways with one copy of its whole pages, :func:`release_requests` gives back the
pages that nobody holds any more, and :func:`compact_pages` moves the live pages
of a pool to its front. All three keep ``holders`` (int32 ``(pages,)``, zeros at
first): how many requests hold a page besides the first. They too read nothing on
the host. Calls on one pool follow one another: on one stream, or ordered by events.
"""

from __future__ import annotations

from collections.abc import Sequence
from typing import NamedTuple

import torch

from kernelo_b200.kernels.attention import _check_index
from kernelo_b200.runtime import native


class StepSlots(NamedTuple):
    """What :func:`build_slots` writes besides the block table."""

    cu_new: torch.Tensor  # int32 (requests + 1,): offsets of each request's added tokens
    positions: torch.Tensor  # int32 (max_tokens,): position of each added token, 0 past the last
    slots: torch.Tensor  # int64 (max_tokens,): page * block + offset, -1 where there is none
    blocks_taken: torch.Tensor  # int32 (1,): pages needed; more than the free list has: it ran out
    dropped: torch.Tensor  # int32 (1,): added tokens that got no slot


def _check(context_lens: torch.Tensor, new_lens: torch.Tensor, block_table: torch.Tensor, free_blocks: torch.Tensor,
           block_size: int, max_tokens: int) -> None:
    if block_size < 1:
        raise ValueError(f"block_size must be positive, got {block_size}")
    if max_tokens < 0:
        raise ValueError(f"max_tokens must not be negative, got {max_tokens}")
    if block_table.ndim != 2 or block_table.dtype != torch.int32:
        raise ValueError(f"block_table must be int32 (requests, blocks), got {block_table.dtype} "
                         f"{tuple(block_table.shape)}")
    if not block_table.is_cuda:
        raise ValueError(f"block_table must be a CUDA tensor, got {block_table.device}")
    if block_table.stride(1) != 1 and block_table.shape[1] > 1:
        raise ValueError("block_table must have contiguous rows")
    seqs = block_table.shape[0]
    for name, t in (("context_lens", context_lens), ("new_lens", new_lens)):
        _check_index(name, t, block_table)
        if t.ndim != 1 or t.shape[0] != seqs:
            raise ValueError(f"{name} must have shape ({seqs},), got {tuple(t.shape)}")
    _check_index("free_blocks", free_blocks, block_table)
    if free_blocks.ndim != 1:
        raise ValueError(f"free_blocks must have one dimension, got shape {tuple(free_blocks.shape)}")


def build_slots(
    context_lens: torch.Tensor,
    new_lens: torch.Tensor,
    block_table: torch.Tensor,
    free_blocks: torch.Tensor,
    *,
    block_size: int,
    max_tokens: int,
) -> StepSlots:
    """Pages and slots for ``new_lens`` tokens added to requests of ``context_lens`` (int32).

    ``block_table`` (int32 ``(requests, blocks)``) holds each request's pages
    so far; the pages a request still needs are taken from ``free_blocks``
    (int32) in order, request after request, and written into its row, -1 where
    the list ends. ``max_tokens`` is the length of ``positions`` and ``slots``
    (at least the sum of ``new_lens``, which only the device knows). The caller
    drops the first ``blocks_taken`` entries of its free list. Called again on
    the same lengths it writes the same values.
    """
    device, seqs = block_table.get_device(), block_table.shape[0]
    # one expression for what is right, and the reasons only where it is not
    if not (block_size > 0 and max_tokens >= 0 and block_table.is_cuda and block_table.ndim == 2
            and block_table.dtype is torch.int32 and block_table.stride(1) == 1
            and context_lens.dtype is torch.int32 and new_lens.dtype is torch.int32 and free_blocks.dtype is torch.int32
            and context_lens.get_device() == device == new_lens.get_device() == free_blocks.get_device()
            and context_lens.ndim == 1 == new_lens.ndim and free_blocks.ndim == 1
            and context_lens.shape[0] == seqs == new_lens.shape[0] and context_lens.is_contiguous()
            and new_lens.is_contiguous() and free_blocks.is_contiguous()):
        _check(context_lens, new_lens, block_table, free_blocks, block_size, max_tokens)
    slots = torch.empty(max_tokens, device=block_table.device, dtype=torch.int64)
    # one buffer for the 32-bit outputs: an allocation or a view costs the host more than the kernel's writes the GPU
    positions, cu_new, taken, dropped = block_table.new_empty(max_tokens + seqs + 3) \
        .split_with_sizes((max_tokens, seqs + 1, 1, 1))
    native.build_slots(context_lens, new_lens, block_table, free_blocks, block_size, cu_new, positions, slots, taken)
    return StepSlots(cu_new, positions, slots, taken, dropped)


MAX_COMPACT_PAGES = 1 << 22


class Forked(NamedTuple):
    """What :func:`fork_requests` reports."""

    blocks_taken: torch.Tensor  # int32 (1,): pages taken; more than the free list has: it ran out
    dropped: torch.Tensor  # int32 (1,): pairs that did nothing, or whose child lacks its last page


class Released(NamedTuple):
    """What :func:`release_requests` gives back."""

    pages: torch.Tensor  # int32 (requests * blocks,): pages that nobody holds any more, -1 behind the last
    count: torch.Tensor  # int32 (1,): how many


class Compacted(NamedTuple):
    """What :func:`compact_pages` has done."""

    renamed: torch.Tensor  # int32 (pages,): each page's new number, -1 for a free page
    live: torch.Tensor  # int32 (1,): live pages, which are the first ones now
    moves: torch.Tensor  # int32 (1,): pages that have moved


def _check_table(block_table: torch.Tensor, context_lens: torch.Tensor, holders: torch.Tensor) -> None:
    if block_table.ndim != 2 or block_table.dtype is not torch.int32:
        raise ValueError(f"block_table must be int32 (requests, blocks), got {block_table.dtype} "
                         f"{tuple(block_table.shape)}")
    if not block_table.is_cuda:
        raise ValueError(f"block_table must be a CUDA tensor, got {block_table.device}")
    rows, cols = block_table.shape
    device = block_table.get_device()
    # one expression for what is right, and the reasons only where it is not
    if (block_table.is_contiguous() and context_lens.dtype is torch.int32 and context_lens.get_device() == device
            and context_lens.shape == (rows,) and context_lens.is_contiguous() and holders.dtype is torch.int32
            and holders.get_device() == device and holders.ndim == 1 and holders.is_contiguous()):
        return
    if (block_table.stride(1) != 1 and cols > 1) or (block_table.stride(0) < cols and rows > 1):
        raise ValueError("block_table must have contiguous rows that do not overlap")
    _check_index("context_lens", context_lens, block_table)
    if context_lens.ndim != 1 or context_lens.shape[0] != rows:
        raise ValueError(f"context_lens must have shape ({rows},), got {tuple(context_lens.shape)}")
    _check_index("holders", holders, block_table)
    if holders.ndim != 1:
        raise ValueError(f"holders must have one dimension, got shape {tuple(holders.shape)}")


def _check_list(name: str, t: torch.Tensor, block_table: torch.Tensor) -> None:
    _check_index(name, t, block_table)
    if t.ndim != 1:
        raise ValueError(f"{name} must have one dimension, got shape {tuple(t.shape)}")


def _check_caches(caches: Sequence[torch.Tensor], block_table: torch.Tensor, holders: torch.Tensor) -> list[torch.Tensor]:
    caches = list(caches)
    if not caches:
        raise ValueError("expected at least one cache")
    first = caches[0]
    shape, stride, dtype, device = first.shape, first.stride(), first.dtype, block_table.get_device()
    if len(shape) != 4 or shape[2] < 1:
        raise ValueError(f"expected caches (pages, kv_heads, block, dim), got {tuple(shape)}")
    if shape[0] != holders.shape[0]:
        raise ValueError(f"holders must have shape ({shape[0]},) for caches {tuple(shape)}, got {tuple(holders.shape)}")
    n = len(caches)
    # all at once (a model has a cache for each layer's keys and values), and one by one where something is wrong
    if not ([c.shape for c in caches].count(shape) == n == [c.stride() for c in caches].count(stride)
            and [c.dtype for c in caches].count(dtype) == n == [c.get_device() for c in caches].count(device)):
        for c in caches:
            if c.shape != shape or c.stride() != stride or c.dtype is not dtype:
                raise ValueError(f"caches must have one type, shape and strides, got {dtype} {tuple(shape)} {stride} and "
                                 f"{c.dtype} {tuple(c.shape)} {c.stride()}")
            if c.get_device() != device:
                raise ValueError(f"caches must be on {block_table.device}, got {c.device}")
    if stride[3] != 1 and shape[3] > 1:
        raise ValueError("caches must have a contiguous last dimension")
    if any(s == 0 and n > 1 for s, n in zip(stride, shape)):
        raise ValueError(f"caches overlap themselves: strides {stride} for shape {tuple(shape)}")
    return caches


def fork_requests(
    caches: Sequence[torch.Tensor],
    block_table: torch.Tensor,
    context_lens: torch.Tensor,
    holders: torch.Tensor,
    free_blocks: torch.Tensor,
    parents: torch.Tensor,
    children: torch.Tensor,
) -> Forked:
    """Row ``children[i]`` becomes a copy of the request in row ``parents[i]`` (int32 both).

    ``caches``: every layer's keys and values ``(pages, kv_heads, block, dim)``, of
    one type, shape and strides. A child holds its parent's whole pages together
    with it; for the tokens of a last, partial page it gets a page of its own
    from ``free_blocks`` (int32), one for each such pair in order, and those tokens
    are copied in all caches. The rest of its row becomes -1, and
    ``context_lens[child]`` its parent's length. So nobody ever writes to a page
    held together: new tokens go behind the last one.

    Children are free rows: all different, and none of them a parent. A pair
    that breaks this, or names a row that is none, does nothing and counts as
    dropped, as does a child whose page the free list lacks (it has -1 there).
    The caller drops the first ``blocks_taken`` entries of its free list.
    """
    _check_table(block_table, context_lens, holders)
    caches = _check_caches(caches, block_table, holders)
    _check_list("free_blocks", free_blocks, block_table)
    _check_list("parents", parents, block_table)
    _check_list("children", children, block_table)
    if parents.shape != children.shape:
        raise ValueError(f"parents and children must have one shape, got {tuple(parents.shape)} and {tuple(children.shape)}")
    counts = block_table.new_empty((2, 1))
    native.fork(caches, block_table, context_lens, holders, free_blocks, parents, children, counts)
    return Forked(*counts.unbind(0))


def release_requests(
    block_table: torch.Tensor,
    context_lens: torch.Tensor,
    holders: torch.Tensor,
    requests: torch.Tensor,
    *,
    block_size: int,
) -> Released:
    """The requests in the rows ``requests`` (int32) end: their rows become -1, their lengths 0.

    Pages that other requests still hold lose a holder; the others come back in
    the order of the list and of their columns (a page of several of these
    requests where the first has it). A row that is named twice ends once; one
    that is none is skipped. The caller appends the first ``count`` of ``pages``
    to its free list.
    """
    _check_table(block_table, context_lens, holders)
    _check_list("requests", requests, block_table)
    if block_size < 1:
        raise ValueError(f"block_size must be positive, got {block_size}")
    n, cols = requests.shape[0], block_table.shape[1]
    parts = n * -(-cols // 256)
    if parts > 200_000 or n * cols >= 1 << 30:
        raise ValueError(f"requests of one call must have 200000 parts of 256 blocks at most, got {n} x {cols}")
    scratch, pages, count = block_table.new_empty(9 * parts + n * cols + 1).split_with_sizes((9 * parts, n * cols, 1))
    native.release(block_table, context_lens, holders, requests, block_size, scratch, pages, count)
    return Released(pages, count)


def compact_pages(
    caches: Sequence[torch.Tensor],
    block_table: torch.Tensor,
    context_lens: torch.Tensor,
    holders: torch.Tensor,
) -> Compacted:
    """Moves the live pages of a pool to its front, in all ``caches`` (as in :func:`fork_requests`).

    Live are the pages of the tokens that the requests have. With ``live`` of them,
    those numbered ``live`` and above go, in order, to the free places below;
    the block table and ``holders`` follow. What the pool holds is then its first
    ``live`` pages, and its free list ``live, live + 1, ..``. Slots and page
    numbers taken before are stale: ``renamed`` translates them.
    """
    _check_table(block_table, context_lens, holders)
    caches = _check_caches(caches, block_table, holders)
    pages = holders.shape[0]
    if pages > MAX_COMPACT_PAGES:
        raise ValueError(f"compact_pages takes pools of at most {MAX_COMPACT_PAGES} pages, got {pages}")
    renamed, sources, targets, live, moves = block_table.new_empty(pages + 2 * (pages // 2) + 2) \
        .split_with_sizes((pages, pages // 2, pages // 2, 1, 1))
    native.compact(caches, block_table, context_lens, holders, renamed, sources, targets, live)
    return Compacted(renamed, live, moves)

"""Pages of a key/value cache, and the plan of a serving step built on the GPU.

:func:`build_slots` takes the lengths of a batch's requests and writes, in one
launch, everything that the step's other calls read: new pages into the block
table, and the offset, position and cache slot of every added token. Nothing is
read on the host, so it can be captured with the step.
"""

from __future__ import annotations

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

"""Rotary positions on sm_100a, with the paged cache's write fused in.

The first ``rot`` elements of each head are turned pair by pair by the angle of
the token's position: pairs ``(i, i + rot/2)``, or ``(2i, 2i + 1)`` with
``interleaved=True``; the rest of the head is left as it is. The angles come
from a table that :func:`rotary_table` makes once, in 64 bits, plain or scaled
for contexts longer than a model was trained on. The rotation is orthogonal, so
its gradient is the turn back: ``inverse=True``.
"""

from __future__ import annotations

import math

import torch

from kernelo_b200.kernels.attention import _check_index, _check_operand, _empty_like
from kernelo_b200.runtime import native

SCALINGS = ("linear", "base", "parts")


def rotary_table(
    max_positions: int,
    rotary_dim: int,
    *,
    base: float = 10000.0,
    scaling: str | None = None,
    factor: float = 1.0,
    original_positions: int | None = None,
    low_turns: float = 1.0,
    high_turns: float = 32.0,
    device: torch.device | str = "cuda",
) -> torch.Tensor:
    """cos and sin of every position: fp32 ``(max_positions, rotary_dim)``, cosines first.

    Pair ``i`` turns by ``position * base ** (-2 i / rotary_dim)``. ``scaling``
    stretches the table to ``factor`` times the trained context:

    * ``"linear"`` -- positions divided by ``factor``;
    * ``"base"`` -- ``base`` raised by ``factor ** (rotary_dim / (rotary_dim - 2))``,
      which divides the slowest pair's frequency by ``factor`` and leaves the fastest;
    * ``"parts"`` -- pairs that turn at least ``high_turns`` times within
      ``original_positions`` keep their frequency, those that turn at most
      ``low_turns`` times have it divided by ``factor``, the ones between are
      blended linearly in their number of turns.
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and positive, got {rotary_dim}")
    if max_positions < 0:
        raise ValueError(f"max_positions must not be negative, got {max_positions}")
    if scaling is not None and scaling not in SCALINGS:
        raise ValueError(f"scaling must be None or one of {SCALINGS}, got {scaling!r}")
    if scaling is not None and not factor >= 1.0:
        raise ValueError(f"factor must be at least 1, got {factor}")
    if scaling == "base":
        if rotary_dim == 2:
            raise ValueError("scaling 'base' needs at least two pairs")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    frequency = base ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim)
    if scaling == "linear":
        frequency = frequency / factor
    elif scaling == "parts":
        if original_positions is None or not high_turns > low_turns:
            raise ValueError("scaling 'parts' needs original_positions and high_turns > low_turns")
        turns = original_positions * frequency / (2 * math.pi)
        keep = ((turns - low_turns) / (high_turns - low_turns)).clamp(0.0, 1.0)
        frequency = frequency * (keep + (1.0 - keep) / factor)
    angle = torch.arange(max_positions, dtype=torch.float64, device=device)[:, None] * frequency
    return torch.cat([angle.cos(), angle.sin()], dim=1).float()


def _check(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, table: torch.Tensor) -> None:
    device = q.get_device()
    # one expression for what is right, and the reasons only where it is not
    if (q.is_cuda and q.ndim == 3 == k.ndim and k.dtype is q.dtype and q.shape[0] == k.shape[0]
            and q.shape[2] == k.shape[2] and q.stride(2) == 1 == k.stride(2) and k.get_device() == device
            and positions.dtype is torch.int32 and positions.get_device() == device and positions.ndim == 1
            and positions.shape[0] == q.shape[0] and positions.is_contiguous()
            and table.dtype is torch.float32 and table.get_device() == device and table.ndim == 2
            and table.is_contiguous() and table.shape[1] <= q.shape[2] and table.shape[1] % 2 == 0):
        return
    if q.ndim != 3 or k.ndim != 3 or q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2]:
        raise ValueError("expected q (tokens, heads, dim) and k (tokens, kv_heads, dim), got "
                         f"{tuple(q.shape)} and {tuple(k.shape)}")
    if not q.is_cuda:
        raise ValueError(f"q must be a CUDA tensor, got {q.device}")
    _check_operand("q", q, q)
    _check_operand("k", k, q)
    _check_index("positions", positions, q)
    if positions.ndim != 1 or positions.shape[0] != q.shape[0]:
        raise ValueError(f"positions must have shape ({q.shape[0]},), got {tuple(positions.shape)}")
    _check_index("table", table, q, torch.float32)
    if table.ndim != 2 or table.shape[1] % 2 or table.shape[1] > q.shape[2]:
        raise ValueError(f"table must be (positions, rotary_dim) with an even rotary_dim of at most {q.shape[2]}, "
                         f"got {tuple(table.shape)}")


def _check_cache(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                 slots: torch.Tensor) -> None:
    if v.shape != k.shape:
        raise ValueError(f"v must have k's shape {tuple(k.shape)}, got {tuple(v.shape)}")
    _check_operand("v", v, q)
    if k_cache.ndim != 4 or k_cache.shape != v_cache.shape or k_cache.shape[1] != k.shape[1] \
            or k_cache.shape[3] != k.shape[2] or k_cache.shape[2] < 1:
        raise ValueError(f"expected caches (pages, {k.shape[1]}, block, {k.shape[2]}), got {tuple(k_cache.shape)} "
                         f"and {tuple(v_cache.shape)}")
    _check_operand("k_cache", k_cache, q)
    _check_operand("v_cache", v_cache, q)
    _check_index("slots", slots, q, torch.int64)
    if slots.ndim != 1 or slots.shape[0] != q.shape[0]:
        raise ValueError(f"slots must have shape ({q.shape[0]},), got {tuple(slots.shape)}")


def _output(name: str, out: torch.Tensor | None, like: torch.Tensor) -> torch.Tensor:
    if out is None:
        return _empty_like(like)
    if out is not like:
        if out.shape != like.shape:
            raise ValueError(f"{name} must have shape {tuple(like.shape)}, got {tuple(out.shape)}")
        _check_operand(name, out, like)
    return out


def rotary(
    q: torch.Tensor,
    k: torch.Tensor,
    positions: torch.Tensor,
    table: torch.Tensor,
    *,
    interleaved: bool = False,
    inverse: bool = False,
    q_out: torch.Tensor | None = None,
    k_out: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """q ``(tokens, heads, dim)`` and k ``(tokens, kv_heads, dim)`` turned by ``positions`` (int32).

    ``q_out`` / ``k_out`` may be q and k themselves. A position outside the
    table gives NaN. ``inverse=True`` turns back: the gradient of the outputs
    goes in, that of the inputs comes out.
    """
    _check(q, k, positions, table)
    q_out, k_out = _output("q_out", q_out, q), _output("k_out", k_out, k)
    if q.numel() or k.numel():
        native.rotary(q, k, q_out, k_out, positions, table, interleaved=interleaved, inverse=inverse)
    return q_out, k_out


def rotary_to_cache(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    positions: torch.Tensor,
    table: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    slots: torch.Tensor,
    *,
    interleaved: bool = False,
    q_out: torch.Tensor | None = None,
    k_out: torch.Tensor | None = None,
) -> torch.Tensor:
    """:func:`rotary`, with the turned k and v written to their cache slots.

    ``slots`` (int64 ``(tokens,)``) are ``page * block + offset`` into caches
    ``(pages, kv_heads, block, dim)``; a negative one is not written. Returns
    the turned q; the turned k is also written to ``k_out`` when given (a
    prompt's attention reads it packed). Two tokens with one slot: either may
    end up in it.
    """
    _check(q, k, positions, table)
    dtype, device = q.dtype, q.get_device()
    if not (v.shape == k.shape and v.dtype is dtype and v.get_device() == device and v.stride(2) == 1
            and k_cache.ndim == 4 and v_cache.shape == k_cache.shape and k_cache.shape[1] == k.shape[1]
            and k_cache.shape[3] == k.shape[2] and k_cache.shape[2] > 0 and k_cache.dtype is dtype
            and v_cache.dtype is dtype and k_cache.get_device() == device == v_cache.get_device()
            and k_cache.stride(3) == 1 == v_cache.stride(3) and slots.dtype is torch.int64
            and slots.get_device() == device and slots.ndim == 1 and slots.shape[0] == q.shape[0]
            and slots.is_contiguous()):
        _check_cache(q, k, v, k_cache, v_cache, slots)
    q_out = _output("q_out", q_out, q)
    if k_out is not None:
        k_out = _output("k_out", k_out, k)
    if q.numel() or k.numel():
        native.rotary(q, k, q_out, k_out, positions, table, interleaved=interleaved, inverse=False, v=v,
                      k_cache=k_cache, v_cache=v_cache, slots=slots)
    return q_out

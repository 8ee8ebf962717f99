"""Rotary positions on sm_100a, with the paged cache's write fused in.

The first ``rot`` elements of each head are turned pair by pair by the angle of
the token's position: pairs ``(i, i + rot/2)``, or ``(2i, 2i + 1)`` with
``interleaved=True``; the rest of the head is left as it is. The angles come
from a table that :func:`rotary_table` makes once, in 64 bits, plain or scaled
for contexts longer than a model was trained on. The rotation is orthogonal, so
its gradient is the turn back: ``inverse=True``.

Models that normalise each head of q and k before the turn do both in one pass
with :func:`norm_rotary` and :func:`norm_rotary_to_cache`, and have the gradient
of both from :func:`norm_rotary_backward`.
"""

from __future__ import annotations

import math

import torch

from kernelo_b200.kernels.attention import _check_index, _check_operand, _check_output, _empty_like
from kernelo_b200.kernels.rmsnorm import DEFAULT_EPS
from kernelo_b200.runtime import native

SCALINGS = ("linear", "base", "parts")
MAX_NORM_DIM = 256
_EPS_RANGE = torch.finfo(torch.float32).tiny, torch.finfo(torch.float32).max


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
    device, shape, k_shape, turned = q.get_device(), q.shape, k.shape, table.shape
    # one expression for what is right, and the reasons only where it is not
    if (q.is_cuda and len(shape) == 3 == len(k_shape) and k.dtype is q.dtype and shape[0] == k_shape[0]
            and shape[2] == k_shape[2] and q.stride()[2] == 1 == k.stride()[2] and k.get_device() == device
            and positions.dtype is torch.int32 and positions.get_device() == device and positions.ndim == 1
            and positions.shape[0] == shape[0] and positions.is_contiguous()
            and table.dtype is torch.float32 and table.get_device() == device and len(turned) == 2
            and table.is_contiguous() and turned[1] <= shape[2] and turned[1] % 2 == 0):
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


def _check_cached(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                  slots: torch.Tensor) -> None:
    dtype, device, k_shape, pages = q.dtype, q.get_device(), k.shape, k_cache.shape
    if not (v.shape == k_shape and v.dtype is dtype and v.get_device() == device and v.stride()[2] == 1
            and len(pages) == 4 and v_cache.shape == pages and pages[1] == k_shape[1] and pages[3] == k_shape[2]
            and pages[2] > 0 and k_cache.dtype is dtype and v_cache.dtype is dtype
            and k_cache.get_device() == device == v_cache.get_device()
            and k_cache.stride()[3] == 1 == v_cache.stride()[3] and slots.dtype is torch.int64
            and slots.get_device() == device and slots.ndim == 1 and slots.shape[0] == k_shape[0]
            and slots.is_contiguous()):
        _check_cache(q, k, v, k_cache, v_cache, slots)


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
    _check_cached(q, k, v, k_cache, v_cache, slots)
    q_out = _output("q_out", q_out, q)
    if k_out is not None:
        k_out = _output("k_out", k_out, k)
    if q.numel() or k.numel():
        native.rotary(q, k, q_out, k_out, positions, table, interleaved=interleaved, inverse=False, v=v,
                      k_cache=k_cache, v_cache=v_cache, slots=slots)
    return q_out


def _check_norm(q: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, eps: float) -> None:
    shape, dtype, device = q.shape[2:], q.dtype, q.get_device()
    # one expression for what is right, and the reasons only where it is not
    if (q_weight.shape == shape == k_weight.shape and q_weight.dtype is dtype and k_weight.dtype is dtype
            and q_weight.get_device() == device == k_weight.get_device() and q_weight.is_contiguous()
            and k_weight.is_contiguous() and shape[0] <= MAX_NORM_DIM and _EPS_RANGE[0] <= eps <= _EPS_RANGE[1]):
        return
    if shape[0] > MAX_NORM_DIM:
        raise ValueError(f"norms take heads of at most {MAX_NORM_DIM} elements, got {shape[0]}")
    if not _EPS_RANGE[0] <= eps <= _EPS_RANGE[1]:
        raise ValueError(f"eps must be positive and in fp32's normal range, got {eps}")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w.shape != shape:
            raise ValueError(f"{name} must have shape ({shape[0]},), got {tuple(w.shape)}")
        _check_operand(name, w, q)


def _same_place(a: torch.Tensor, b: torch.Tensor) -> bool:
    return a.data_ptr() == b.data_ptr() and a.shape == b.shape and a.stride() == b.stride()


def _norm_outputs(q: torch.Tensor, k: torch.Tensor, q_out: torch.Tensor | None, k_out: torch.Tensor | None,
                  others: dict[str, torch.Tensor]) -> None:
    """Outputs given by the caller: q and k themselves, or memory that no operand and no other output shares."""
    given = {name: (out, x) for name, out, x in (("q_out", q_out, q), ("k_out", k_out, k)) if out is not None}
    for name, (out, x) in given.items():
        if out.shape != x.shape:
            raise ValueError(f"{name} must have shape {tuple(x.shape)}, got {tuple(out.shape)}")
        _check_operand(name, out, x)
        own = "q" if x is q else "k"
        operands = {"q": q, "k": k, **others}
        if _same_place(out, x):
            del operands[own]
        if name == "k_out" and q_out is not None:
            operands["q_out"] = q_out
        _check_output(name, out, operands)


def norm_rotary(
    q: torch.Tensor,
    k: torch.Tensor,
    positions: torch.Tensor,
    table: torch.Tensor,
    q_weight: torch.Tensor,
    k_weight: torch.Tensor,
    *,
    eps: float = DEFAULT_EPS,
    interleaved: bool = False,
    q_out: torch.Tensor | None = None,
    k_out: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """:func:`rotary` of heads normalised first: each head ``x`` of q and k becomes
    ``weight * x / sqrt(mean(x^2) + eps)`` before its turn.

    ``q_weight`` and ``k_weight`` (``(dim,)``, of the operands' type) are shared
    by the heads of q and those of k; ``eps`` is positive and in fp32's normal
    range. Everything is computed in fp32 and rounded once, so the result is
    nearer than that of a norm and a turn apart. ``q_out`` / ``k_out`` may be q and
    k themselves, and share no other operand's memory.
    """
    _check(q, k, positions, table)
    _check_norm(q, q_weight, k_weight, eps)
    if q_out is not None or k_out is not None:
        _norm_outputs(q, k, q_out, k_out, {})
    q_out = _empty_like(q) if q_out is None else q_out
    k_out = _empty_like(k) if k_out is None else k_out
    if q.numel() or k.numel():
        native.norm_rotary(q, k, q_out, k_out, positions, table, q_weight, k_weight, eps, interleaved=interleaved)
    return q_out, k_out


def norm_rotary_to_cache(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    positions: torch.Tensor,
    table: torch.Tensor,
    q_weight: torch.Tensor,
    k_weight: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    slots: torch.Tensor,
    *,
    eps: float = DEFAULT_EPS,
    interleaved: bool = False,
    q_out: torch.Tensor | None = None,
    k_out: torch.Tensor | None = None,
) -> torch.Tensor:
    """:func:`rotary_to_cache` of heads normalised first, as :func:`norm_rotary` does; v is written as it is.

    The caches share no memory with an operand or with each other (keys and values may lie in turn in one buffer)."""
    _check(q, k, positions, table)
    _check_cached(q, k, v, k_cache, v_cache, slots)
    _check_norm(q, q_weight, k_weight, eps)
    if q_out is not None or k_out is not None:
        _norm_outputs(q, k, q_out, k_out, {"v": v, "k_cache": k_cache, "v_cache": v_cache})
    q_out = _empty_like(q) if q_out is None else q_out
    if q.numel() or k.numel():
        native.norm_rotary(q, k, q_out, k_out, positions, table, q_weight, k_weight, eps, interleaved=interleaved, v=v,
                           k_cache=k_cache, v_cache=v_cache, slots=slots)
    return q_out


def norm_rotary_backward(
    dq: torch.Tensor,
    dk: torch.Tensor,
    q: torch.Tensor,
    k: torch.Tensor,
    positions: torch.Tensor,
    table: torch.Tensor,
    q_weight: torch.Tensor,
    k_weight: torch.Tensor,
    *,
    eps: float = DEFAULT_EPS,
    interleaved: bool = False,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """Gradients of q, k, ``q_weight`` and ``k_weight``, given those of :func:`norm_rotary`'s outputs and its inputs.

    The weights' gradients are fp32 sums over all tokens and heads, added in a
    fixed order: a call on the same operands gives the same bits. A token whose
    position the table lacks makes them NaN.
    """
    _check(q, k, positions, table)
    _check_norm(q, q_weight, k_weight, eps)
    dtype, device = q.dtype, q.get_device()
    if not (dq.shape == q.shape and dk.shape == k.shape and dq.dtype is dtype and dk.dtype is dtype
            and dq.get_device() == device == dk.get_device() and dq.stride(2) == 1 == dk.stride(2)):
        for name, d, x in (("dq", dq, q), ("dk", dk, k)):
            if d.shape != x.shape:
                raise ValueError(f"{name} must have shape {tuple(x.shape)}, got {tuple(d.shape)}")
            _check_operand(name, d, q)
    q_grad, k_grad, dim = _empty_like(q), _empty_like(k), q.shape[2]
    weight_grads = table.new_empty(2, dim)
    if dim:
        native.norm_rotary_grad(dq, dk, q, k, q_grad, k_grad, positions, table, q_weight, k_weight, eps, weight_grads,
                                interleaved=interleaved)
    return q_grad, k_grad, *weight_grads.unbind(0)

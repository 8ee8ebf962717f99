"""Attention for serving on sm_100a: whole prompts, and new tokens over a paged cache.

``o = softmax(scale * q k^T) v`` per head, scores and softmax statistics in
fp32, grouped heads read in place (query head ``h`` uses key head
``h // (heads // kv_heads)``). The reference leaves attention to PyTorch
(``kernelforge/integration/transformer.py:71-187``); these are what its block
needs once prompts have different lengths and keys live in pages.

* :func:`prefill_attention` -- prompts packed without padding, causal or not.
* :func:`tree_attention` -- one token or a tree of drafted tokens per request
  over a paged cache.

Lengths and offsets stay on the device: no call reads them on the host, so both
can be captured in a CUDA graph and replayed with other lengths. A row that
sees no key gives zeros (log-sum-exp ``-inf``), and what a row does not see
never reaches it, whatever is stored there. A score that is NaN or +infinity
makes the rows that see it NaN, log-sum-exp included.
"""

from __future__ import annotations

import torch

from kernelo_b200.runtime import native

MAX_HEAD_DIM = 256


def _check_heads(q: torch.Tensor, kv_heads: int, dim: int) -> None:
    if q.shape[2] != dim:
        raise ValueError(f"head dimension mismatch: q {tuple(q.shape)} against keys of {dim}")
    if dim > MAX_HEAD_DIM:
        raise ValueError(f"attention takes heads of at most {MAX_HEAD_DIM} elements, got {dim}")
    if q.shape[1] % kv_heads if kv_heads else q.shape[1]:
        raise ValueError(f"{q.shape[1]} query heads are not a multiple of {kv_heads} key heads")


def _check_operand(name: str, t: torch.Tensor, q: torch.Tensor) -> None:
    if t.dtype is not q.dtype:
        raise ValueError(f"dtype mismatch: {q.dtype} vs {name} {t.dtype}")
    if t.get_device() != q.get_device():
        raise ValueError(f"{name} must be on one device with the first operand, got {t.device} and {q.device}")
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"{name} must have a contiguous last dimension. Pass {name}.contiguous() explicitly.")


def _check_index(name: str, t: torch.Tensor, q: torch.Tensor, dtype: torch.dtype = torch.int32) -> None:
    if t.dtype is not dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if t.get_device() != q.get_device():
        raise ValueError(f"{name} must be on {q.device}, got {t.device}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _empty_like(t: torch.Tensor) -> torch.Tensor:
    """A contiguous tensor of t's shape (empty_like is the cheaper call, but keeps a view's order)."""
    if t.is_contiguous():
        return torch.empty_like(t)
    return torch.empty(t.shape, device=t.device, dtype=t.dtype)


def _elements(t: torch.Tensor) -> int:
    """From the first element to the last, whatever lies between."""
    return sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1 if t.numel() else 0


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors of one type share an element: exact for views of equal strides (the parts of one
    projection, say), and true for others whose address ranges meet."""
    size, delta = a.element_size(), b.data_ptr() - a.data_ptr()
    if not a.numel() or not b.numel() or delta >= _elements(a) * size or -delta >= _elements(b) * size:
        return False
    dims = sorted(zip(a.stride(), b.stride(), a.shape, b.shape), reverse=True) if a.ndim == b.ndim else None
    if dims is None or delta % size or any(s != r and (n > 1 or m > 1) for s, r, n, m in dims):
        return True

    def meet(delta, dims):  # sum of i s over the dimensions is delta for some i > -m and < n in each
        if not dims:
            return delta == 0
        (s, _, n, m), rest = dims[0], dims[1:]
        if s == 0 or n == m == 1:
            return meet(delta, rest)
        low, high = -sum((d[3] - 1) * d[0] for d in rest), sum((d[2] - 1) * d[0] for d in rest)
        first, last = max(1 - m, -((high - delta) // s)), min(n - 1, (delta - low) // s)
        return last - first > 64 or any(meet(delta - i * s, rest) for i in range(first, last + 1))

    return meet(delta // size, dims)


def _check_output(name: str, out: torch.Tensor, operands: dict[str, torch.Tensor]) -> None:
    """An output written by many threads, beside others that still read, shares no element with itself or them."""
    span = 0
    for s, n in sorted((s, n) for s, n in zip(out.stride(), out.shape) if n > 1):
        if s <= span:
            raise ValueError(f"{name} overlaps itself: strides {out.stride()} for shape {tuple(out.shape)}")
        span += (n - 1) * s
    for other, t in operands.items():
        if _overlap(out, t):
            raise ValueError(f"{name} shares memory with {other}")


def _check_query(q: torch.Tensor) -> None:
    if q.ndim != 3:
        raise ValueError(f"expected q as (rows, heads, dim), got shape {tuple(q.shape)}")
    if not q.is_cuda:
        raise ValueError(f"q must be a CUDA tensor, got {q.device}")
    if q.stride(2) != 1 and q.shape[2] > 1:
        raise ValueError("q must have a contiguous last dimension. Pass q.contiguous() explicitly.")


def _check_given(out: torch.Tensor, q: torch.Tensor, operands: dict[str, torch.Tensor]) -> None:
    if out.shape != q.shape:
        raise ValueError(f"out must have shape {tuple(q.shape)}, got {tuple(out.shape)}")
    _check_operand("out", out, q)
    _check_output("out", out, operands)


def _outputs(q: torch.Tensor, out: torch.Tensor | None, return_lse: bool):
    if out is None:
        out = _empty_like(q)
    lse = torch.empty(q.shape[0], q.shape[1], device=q.device, dtype=torch.float32) if return_lse else None
    return out, lse


def _check_prefill(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_q: torch.Tensor,
                   cu_k: torch.Tensor | None) -> torch.Tensor:
    _check_query(q)
    if k.ndim != 3 or v.shape != k.shape:
        raise ValueError(f"expected k and v as (keys, kv_heads, dim), got {tuple(k.shape)} and {tuple(v.shape)}")
    _check_operand("k", k, q)
    _check_operand("v", v, q)
    _check_index("cu_q", cu_q, q)
    if cu_q.ndim != 1 or cu_q.shape[0] < 1:
        raise ValueError(f"cu_q must have shape (requests + 1,), got {tuple(cu_q.shape)}")
    if cu_k is None:
        if k.shape[0] != q.shape[0]:
            raise ValueError(f"{k.shape[0]} keys for {q.shape[0]} rows: pass cu_k")
        cu_k = cu_q
    elif cu_k is not cu_q:
        _check_index("cu_k", cu_k, q)
        if cu_k.shape != cu_q.shape:
            raise ValueError(f"cu_q and cu_k must have one shape, got {tuple(cu_q.shape)} and {tuple(cu_k.shape)}")
    return cu_k


def prefill_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    cu_q: torch.Tensor,
    cu_k: torch.Tensor | None = None,
    *,
    causal: bool = True,
    scale: float | None = None,
    out: torch.Tensor | None = None,
    return_lse: bool = False,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """Attention of packed prompts: q ``(rows, heads, dim)``, k and v ``(keys, kv_heads, dim)``.

    ``cu_q`` and ``cu_k`` (int32 ``(requests + 1,)`` on the device, ``cu_k``
    defaulting to ``cu_q``) are the offsets of each request's rows and keys.
    ``causal``: a request's last row sees all of its keys and each row before
    it one less, so a prompt that continues cached keys passes more keys than
    rows. ``scale`` defaults to ``dim ** -0.5``. Returns the output, and with
    ``return_lse`` also the fp32 natural log-sum-exp ``(rows, heads)``. ``out``
    shares no memory with q, k or v.
    """
    dtype, device = q.dtype, q.get_device()
    if cu_k is None and k.shape[:1] == q.shape[:1]:
        cu_k = cu_q
    # one expression for what is right, and the reasons only where it is not: a
    # call costs the host about as long as a short prompt's kernel the GPU
    if not (q.is_cuda and q.ndim == 3 == k.ndim and v.shape == k.shape and cu_k is not None
            and k.dtype is dtype and v.dtype is dtype and k.get_device() == device == v.get_device()
            and q.stride(2) == 1 == k.stride(2) and v.stride(2) == 1
            and cu_q.dtype is torch.int32 and cu_q.get_device() == device and cu_q.ndim == 1 and cu_q.is_contiguous()
            and (cu_k is cu_q or (cu_k.dtype is torch.int32 and cu_k.get_device() == device
                                  and cu_k.shape == cu_q.shape and cu_k.is_contiguous()))):
        cu_k = _check_prefill(q, k, v, cu_q, cu_k)
    _check_heads(q, k.shape[1], k.shape[2])
    if cu_q.shape[0] < 1:
        raise ValueError(f"cu_q must have shape (requests + 1,), got {tuple(cu_q.shape)}")
    if out is not None:
        _check_given(out, q, {"q": q, "k": k, "v": v})
    out, lse = _outputs(q, out, return_lse)
    if q.numel():
        native.prefill_attention(q, k, v, out, lse, cu_q, cu_k, q.shape[2] ** -0.5 if scale is None else scale, causal)
    return (out, lse) if return_lse else out


def _check_tree(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                context_lens: torch.Tensor, cu_q: torch.Tensor | None, tree_mask: torch.Tensor | None) -> None:
    _check_query(q)
    if k_cache.ndim != 4 or v_cache.shape != k_cache.shape:
        raise ValueError("expected k_cache and v_cache as (pages, kv_heads, block, dim), got "
                         f"{tuple(k_cache.shape)} and {tuple(v_cache.shape)}")
    _check_operand("k_cache", k_cache, q)
    _check_operand("v_cache", v_cache, q)
    if block_table.ndim != 2 or block_table.dtype != torch.int32:
        raise ValueError(f"block_table must be int32 (requests, blocks), got {block_table.dtype} "
                         f"{tuple(block_table.shape)}")
    if block_table.get_device() != q.get_device():
        raise ValueError(f"block_table must be on {q.device}, got {block_table.device}")
    if block_table.stride(1) != 1 and block_table.shape[1] > 1:
        raise ValueError("block_table must have contiguous rows")
    seqs = block_table.shape[0]
    _check_index("context_lens", context_lens, q)
    if context_lens.ndim != 1 or context_lens.shape[0] != seqs:
        raise ValueError(f"context_lens must have shape ({seqs},), got {tuple(context_lens.shape)}")
    if cu_q is not None:
        _check_index("cu_q", cu_q, q)
        if cu_q.ndim != 1 or cu_q.shape[0] != seqs + 1:
            raise ValueError(f"cu_q must have shape ({seqs + 1},), got {tuple(cu_q.shape)}")
    elif q.shape[0] != seqs:
        raise ValueError(f"{q.shape[0]} rows for {seqs} requests: pass cu_q")
    if tree_mask is not None:
        _check_index("tree_mask", tree_mask, q, torch.int64)
        if tree_mask.ndim != 2 or tree_mask.shape[0] != q.shape[0] or tree_mask.shape[1] < 1:
            raise ValueError(f"tree_mask must have shape ({q.shape[0]}, words), got {tuple(tree_mask.shape)}")


def tree_attention(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_table: torch.Tensor,
    context_lens: torch.Tensor,
    cu_q: torch.Tensor | None = None,
    tree_mask: torch.Tensor | None = None,
    *,
    scale: float | None = None,
    out: torch.Tensor | None = None,
    return_lse: bool = False,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """Attention of new tokens q ``(rows, heads, dim)`` over pages ``(pages, kv_heads, block, dim)``.

    Position ``i`` of request ``r`` is slot ``i % block`` of page
    ``block_table[r, i // block]`` (int32, -1 for none). Request ``r`` has
    ``context_lens[r]`` cached tokens, seen by all of its rows, followed by its
    own rows' keys and values, written to the cache before the call
    (``rotary_to_cache`` does). ``cu_q`` are the offsets of each request's rows;
    without it every request has one row (plain decoding). ``tree_mask`` (int64
    ``(rows, words)``): bit ``b`` says whether the row sees row ``b`` of its
    request, itself included; without it the rows are a chain. ``out`` shares
    no memory with q or the cache.
    """
    dtype, device = q.dtype, q.get_device()
    if not (q.is_cuda and q.ndim == 3 and k_cache.ndim == 4 and v_cache.shape == k_cache.shape
            and k_cache.dtype is dtype and v_cache.dtype is dtype
            and k_cache.get_device() == device == v_cache.get_device() == block_table.get_device()
            and q.stride(2) == 1 == k_cache.stride(3) and v_cache.stride(3) == 1
            and block_table.ndim == 2 and block_table.dtype is torch.int32 and block_table.stride(1) == 1
            and context_lens.dtype is torch.int32 and context_lens.get_device() == device
            and context_lens.shape == block_table.shape[:1] and context_lens.is_contiguous()
            and cu_q is None and tree_mask is None and q.shape[:1] == context_lens.shape):
        _check_tree(q, k_cache, v_cache, block_table, context_lens, cu_q, tree_mask)
    _check_heads(q, k_cache.shape[1], k_cache.shape[3])
    if k_cache.shape[2] < 1:
        raise ValueError("pages must hold at least one token")
    if out is not None:
        _check_given(out, q, {"q": q, "k_cache": k_cache, "v_cache": v_cache})
    out, lse = _outputs(q, out, return_lse)
    if q.numel():
        native.tree_attention(q, k_cache, v_cache, out, lse, block_table, context_lens, cu_q, tree_mask,
                              q.shape[2] ** -0.5 if scale is None else scale)
    return (out, lse) if return_lse else out

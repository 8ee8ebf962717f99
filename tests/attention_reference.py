"""Attention in 64 bits, and how far a kernel's output may be from it.

The bound is per element and comes from the arithmetic, not from runs: with
``u`` the rounding of the operands' type and ``A_i = sum_j p_ij |v_j|`` (weights
normalised), an output is off by at most

    u |o_i|                                the output's own rounding
  + u A_i                                  the weights rounded for the matrix product
  + 2 A_i (e_s + e_sum)                    scores and sums in fp32

where ``e_s = 4 (D + 8) 2^-24 scale max_j sum_d |q_d k_jd|`` is a fp32 dot product's
error bound in the exponent (4: accumulation that truncates, and the scaling in
base 2), and ``e_sum = 4 (n + 8) 2^-24 + 2^-20`` the sums' over n keys and the exponential's.
16-bit weights below 2^-14 (fp16) have an absolute error of 2^-25 each.
"""

from __future__ import annotations

import math

import torch

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def attend(q, k, v, seen, scale):
    """One head: q (n, D), k and v (m, D), seen (n, m) bool. Output, log-sum-exp and their bounds."""
    unit = UNIT[q.dtype]
    n, dim = q.shape
    keys = k.shape[0]
    q, k, v = q.double(), k.double(), v.double()
    # what no row sees is taken out, whatever it holds; what some row sees is finite in these tests
    used = seen.any(0)
    k = torch.where(used[:, None], k, 0.0)
    v = torch.where(used[:, None], v, 0.0)
    out = torch.zeros(n, dim, dtype=torch.float64, device=q.device)
    lse = torch.full((n,), -math.inf, dtype=torch.float64, device=q.device)
    if keys == 0:
        return out, lse, torch.zeros_like(out), torch.zeros_like(lse)
    scores = torch.where(seen, (q @ k.T) * scale, -math.inf)
    some = seen.any(1)
    top = torch.where(some, scores.amax(1), 0.0)[:, None]
    weights = torch.where(seen, (scores - top).exp(), 0.0)
    sums = weights.sum(1, keepdim=True).clamp(min=1e-300)
    out = (weights / sums) @ v
    lse = torch.where(some, (top + sums.log())[:, 0], lse)
    spread = (weights / sums) @ v.abs()
    magnitude = torch.where(seen, q.abs() @ k.abs().T, 0.0).amax(1, keepdim=True) * abs(scale)
    off_score = 4 * (dim + 8) * 2.0 ** -24 * magnitude
    off_sum = 4 * (keys + 8) * 2.0 ** -24 + 2.0 ** -20
    bound = unit * out.abs() + spread * (unit + 2 * (off_score + off_sum)) + 2.0 ** -40
    if unit == UNIT[torch.float16]:
        bound = bound + 2.0 ** -25 + 2.0 ** -25 * (seen.double() @ v.abs())
    off_lse = (off_score + off_sum)[:, 0] + 2.0 ** -22 * torch.where(some, lse.abs() + top[:, 0].abs(), 0.0)
    return out, lse, bound, off_lse


def check(got, want, bound, what):
    got = got.double()
    assert torch.isfinite(got).all(), f"{what}: {int((~torch.isfinite(got)).sum())} values are not finite"
    over = (got - want).abs() - bound
    worst = float(over.max()) if over.numel() else 0.0
    assert worst <= 0.0, (f"{what}: {int((over > 0).sum())} of {over.numel()} values over their bound, the worst by "
                          f"{worst:.3g} (largest bound {float(bound.max()):.3g})")


def check_lse(got, want, bound, what):
    got = got.double()
    empty = want == -math.inf
    assert torch.equal(got == -math.inf, empty), f"{what}: empty rows differ"
    check(got[~empty], want[~empty], bound[~empty], what + " lse")


def packed(q, k, v, lens_q, lens_k, *, causal=True, scale=None):
    """Reference of packed prompts: out, lse and bounds, rows past the last request zero."""
    scale = q.shape[2] ** -0.5 if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
    off = torch.zeros_like(lse)
    group = q.shape[1] // k.shape[1]
    q0 = k0 = 0
    for n, m in zip(lens_q, lens_k):
        seen = torch.ones(n, m, dtype=torch.bool, device=q.device)
        if causal:
            seen = seen.tril(m - n)
        for h in range(q.shape[1] if n else 0):
            rows, keys = slice(q0, q0 + n), slice(k0, k0 + m)
            out[rows, h], lse[rows, h], bound[rows, h], off[rows, h] = attend(
                q[rows, h], k[keys, h // group], v[keys, h // group], seen, scale)
        q0, k0 = q0 + n, k0 + m
    return out, lse, bound, off


def paged(q, k_cache, v_cache, table, context, nodes, masks=None, *, scale=None):
    """Reference over a paged cache; ``masks``: per request a bool (nodes, nodes) tensor, or None for chains."""
    scale = q.shape[2] ** -0.5 if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
    off = torch.zeros_like(lse)
    group, block = q.shape[1] // k_cache.shape[1], k_cache.shape[2]
    q0 = 0
    for r, (c, n) in enumerate(zip(context, nodes)):
        at = torch.arange(c + n, device=q.device)
        column = at // block
        page = torch.where(column < table.shape[1], table[r].long()[column.clamp(max=table.shape[1] - 1)], -1)
        here = (page >= 0) & (page < k_cache.shape[0])
        k, v = k_cache[page * here, :, at % block], v_cache[page * here, :, at % block]
        seen = torch.ones(n, c + n, dtype=torch.bool, device=q.device)
        seen[:, c:] = masks[r].to(q.device) if masks is not None else seen[:, c:].tril()
        seen &= here
        rows = slice(q0, q0 + n)
        for h in range(q.shape[1] if n else 0):
            out[rows, h], lse[rows, h], bound[rows, h], off[rows, h] = attend(
                q[rows, h], k[:, h // group], v[:, h // group], seen, scale)
        q0 += n
    return out, lse, bound, off

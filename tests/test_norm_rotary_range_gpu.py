"""Head norms of heads whose squares just leave fp32, beside ordinary ones in the same warp, against 64 bits.

Bounds as in ``test_norm_rotary_gpu``: taking elements by a power of two less is exact, and ``eps`` is taken by its square
less with them, which moves the mean by a rounding at most.
"""

from __future__ import annotations

import pytest
import torch

from kernelo_b200.kernels.rotary import norm_rotary, norm_rotary_backward, norm_rotary_to_cache, rotary_table
from tests.test_norm_rotary_gpu import check, check_gradient

pytestmark = pytest.mark.gpu


def large_heads(dim, dtype, device):
    """q and k with a token for each power of two from 2^56 to 2^77: heads of equal, of mixed and of one large element, and
    ordinary ones."""
    gen = torch.Generator().manual_seed(0)
    size = 2.0 ** torch.arange(56, 78, dtype=torch.float64)[:, None, None]
    ordinary = torch.randn(22, 2, dim, generator=gen, dtype=torch.float64)
    equal = torch.full((22, 1, dim), 1.25, dtype=torch.float64) * size
    mixed = torch.randn(22, 1, dim, generator=gen, dtype=torch.float64) * size
    single = torch.zeros(22, 1, dim, dtype=torch.float64)
    single[:, 0, dim // 3] = -1.5
    single[:, 0, dim // 2] = 2.0 ** -60
    q = torch.cat([equal, mixed, ordinary[:, :1], single * size], 1)
    k = torch.cat([ordinary[:, 1:], -equal], 1)
    return q.to(dtype).to(device), k.to(dtype).to(device)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("eps", [1e-6, 1e-5, 1e36])
@pytest.mark.parametrize("dim", [32, 64, 128, 250, 256])
def test_heads_whose_squares_just_leave_fp32(dim, eps, dtype, device):
    q, k = large_heads(dim, dtype, device)
    gen = torch.Generator().manual_seed(1)
    qw, kw = ((torch.randn(dim, generator=gen) * 0.3 + 1).to(dtype).to(device) for _ in range(2))
    table = rotary_table(40, dim, device=device)
    positions = torch.arange(22, dtype=torch.int32, device=device)
    y, z = norm_rotary(q, k, positions, table, qw, kw, eps=eps)
    check(y, q, qw, positions, table, False, eps)
    check(z, k, kw, positions, table, False, eps)
    caches = [torch.zeros(2, 2, 16, dim, device=device, dtype=dtype) for _ in range(2)]
    slots = torch.arange(22, device=device)
    again = norm_rotary_to_cache(q, k, k, positions, table, qw, kw, *caches, slots, eps=eps)
    assert torch.equal(again, y) and torch.equal(caches[0][slots // 16, :, slots % 16], z)
    dq, dk = (torch.randn(x.shape, generator=gen).to(dtype).to(device) for x in (q, k))
    gq, gk, gqw, gkw = norm_rotary_backward(dq, dk, q, k, positions, table, qw, kw, eps=eps)
    check_gradient(gq, gqw, dq, q, qw, positions, table, False, eps)
    check_gradient(gk, gkw, dk, k, kw, positions, table, False, eps)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_heads_of_zeros_and_of_the_least_eps(dtype, device):
    """Squares beside the least normal eps are off by 2^-150 each, a rounding of their mean with it."""
    eps, dim = 2.0 ** -126, 64
    gen = torch.Generator().manual_seed(0)
    q, k, dq, dk = (torch.randn(9, n, dim, generator=gen) for n in (3, 2, 3, 2))
    q[:, 1] *= 2.0 ** -63  # (zeros in fp16)
    q[:, 2], k[:, 1] = 0.0, 0.0
    q, k, dq, dk = (x.to(dtype).to(device) for x in (q, k, dq, dk))
    if dtype == torch.float16:  # the gradient of a head of zeros is 2^63 times as large as what goes in
        dq, dk = dq.clone(), dk.clone()
        dq[:, 1:], dk[:, 1] = 0.0, 0.0
    w = torch.ones(dim, dtype=dtype, device=device)
    table = rotary_table(9, dim, device=device)
    positions = torch.arange(9, dtype=torch.int32, device=device)
    y, z = norm_rotary(q, k, positions, table, w, w, eps=eps)
    check(y, q, w, positions, table, False, eps)
    check(z, k, w, positions, table, False, eps)
    assert not y[:, 2].any() and not z[:, 1].any()
    gq, gk, gqw, gkw = norm_rotary_backward(dq, dk, q, k, positions, table, w, w, eps=eps)
    check_gradient(gq, gqw, dq, q, w, positions, table, False, eps)
    check_gradient(gk, gkw, dk, k, w, positions, table, False, eps)

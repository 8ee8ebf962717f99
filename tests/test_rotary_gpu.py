"""Rotary positions and the cache write, against 64 bits.

A turned element is a c - b s in fp32 rounded once: off by at most
2^-23 (|a c| + |b s|) and half a unit of its type.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from kernelo_b200.kernels.rotary import rotary, rotary_table, rotary_to_cache

pytestmark = pytest.mark.gpu

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
DTYPES = tuple(UNIT)


def turned(x, positions, table, interleaved, inverse=False):
    """The definition on complex numbers in 64 bits, and the bound of each element."""
    rot = table.shape[1]
    row = table.double()[positions.long()][:, None]
    cos, sin = row[..., :rot // 2], row[..., rot // 2:] * (-1 if inverse else 1)
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    xd, y = x.double(), x.double().clone()
    y[..., a] = xd[..., a] * cos - xd[..., b] * sin
    y[..., b] = xd[..., a] * sin + xd[..., b] * cos
    bound = torch.zeros_like(y)
    bound[..., a] = xd[..., a].abs() * cos.abs() + xd[..., b].abs() * sin.abs()
    bound[..., b] = xd[..., a].abs() * sin.abs() + xd[..., b].abs() * cos.abs()
    return y, 2.0 ** -23 * bound + UNIT[x.dtype] * y.abs() + (2.0 ** -25 if x.dtype == torch.float16 else 2.0 ** -140)


def check(got, x, positions, table, interleaved, inverse=False):
    want, bound = turned(x, positions, table, interleaved, inverse)
    assert ((got.double() - want).abs() <= bound).all()
    rot = table.shape[1]
    assert torch.equal(got[..., rot:], x[..., rot:])


def inputs(tokens, heads, kv_heads, dim, dtype, device, most=5000, seed=0):
    gen = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(tokens, h, dim, generator=gen).to(dtype).to(device) for h in (heads, kv_heads, kv_heads))
    return q, k, v, torch.randint(0, most, (tokens,), generator=gen, dtype=torch.int32).to(device)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rot", [(128, 128), (128, 64), (64, 64), (80, 80), (80, 40), (80, 20), (96, 24), (20, 6),
                                     (36, 32), (7, 4), (256, 256), (64, 2)])
def test_layouts_and_parts(dim, rot, interleaved, dtype, device):
    q, k, _, positions = inputs(37, 5, 3, dim, dtype, device)
    table = rotary_table(5000, rot, device=device)
    got = rotary(q, k, positions, table, interleaved=interleaved)
    check(got[0], q, positions, table, interleaved)
    check(got[1], k, positions, table, interleaved)
    back = rotary(q, k, positions, table, interleaved=interleaved, inverse=True)
    check(back[0], q, positions, table, interleaved, True)
    check(back[1], k, positions, table, interleaved, True)


@pytest.mark.parametrize("tokens,heads,kv_heads", [(1, 1, 1), (1, 32, 8), (3, 7, 1), (1000, 8, 8), (4097, 4, 2)])
def test_sizes(tokens, heads, kv_heads, device):
    q, k, _, positions = inputs(tokens, heads, kv_heads, 128, torch.bfloat16, device)
    table = rotary_table(5000, 128, device=device)
    for x, y in zip((q, k), rotary(q, k, positions, table)):
        check(y, x, positions, table, False)
    assert rotary(q[:0], k[:0], positions[:0], table)[0].shape == (0, heads, 128)


@pytest.mark.parametrize("dtype", DTYPES)
def test_views_in_place_and_odd_strides(dtype, device):
    qkv = torch.randn(65, 12, 64, device=device).to(dtype)
    positions = torch.arange(65, dtype=torch.int32, device=device)
    table = rotary_table(65, 32, device=device)
    q, k = qkv[:, :8], qkv[:, 8:10]
    before, rest = qkv.clone(), qkv[:, 10:].clone()
    a, b = rotary(q, k, positions, table)
    got = rotary(q, k, positions, table, q_out=q, k_out=k)
    assert got[0] is q and torch.equal(q, a) and torch.equal(k, b) and torch.equal(qkv[:, 10:], rest)
    check(q, before[:, :8], positions, table, False)
    odd = torch.randn(65, 5, 67, device=device).to(dtype)
    q, k = odd[:, :4, 1:65], odd[:, 4:, 3:67]
    for interleaved in (False, True):
        for x, y in zip((q, k), rotary(q, k, positions, table, interleaved=interleaved)):
            check(y, x, positions, table, interleaved)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient(interleaved, dtype, device):
    """The turn back is the gradient: <w, R x> has the gradient R^T w, by the
    formula and by differences (the map is linear, so a difference is exact up
    to the roundings of two outputs)."""
    q, k, _, positions = inputs(9, 3, 3, 32, dtype, device)
    table = rotary_table(5000, 24, device=device)
    w = torch.randn(9, 3, 32, device=device).to(dtype)
    grad = rotary(w, w, positions, table, interleaved=interleaved, inverse=True)[0]
    step = torch.zeros(9, 3, 32, device=device, dtype=dtype)
    for e in range(32):
        step.zero_()
        step[..., e] = 1.0
        up = rotary(step, step, positions, table, interleaved=interleaved)[0]
        down = rotary(-step, -step, positions, table, interleaved=interleaved)[0]
        slope = ((up.double() - down.double()) / 2 * w.double()).sum(-1)
        # two entries of magnitude at most one, each rounded, times w, and the gradient's rounding
        bound = 2 * UNIT[dtype] * w.double().abs().sum(-1) + UNIT[dtype] * grad[..., e].double().abs() + 2.0 ** -20
        assert ((grad[..., e].double() - slope).abs() <= bound).all()
    there = rotary(q, k, positions, table, interleaved=interleaved)
    back = rotary(*there, positions, table, interleaved=interleaved, inverse=True)[0]
    size = (q.double()[..., :24].abs().amax() * 2 + 1)
    assert ((back.double() - q.double()).abs() <= 4 * UNIT[dtype] * size + 2.0 ** -20).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,rot,block", [(128, 128, 16), (64, 32, 24), (20, 6, 5)])
@pytest.mark.parametrize("keep", [False, True])
def test_cache_write(dim, rot, block, keep, dtype, device):
    tokens = 50
    q, k, v, positions = inputs(tokens, 6, 2, dim, dtype, device)
    table = rotary_table(5000, rot, device=device)
    k_cache = torch.full((9 + 50 // block, 2, block, dim), 5.0, device=device, dtype=dtype)
    v_cache = torch.full_like(k_cache, 6.0)
    places = np.random.default_rng(0).permutation(k_cache.shape[0] * block)[:tokens]
    slots = torch.from_numpy(places).to(device)
    slots[3], slots[7], slots[9] = -1, k_cache.shape[0] * block, 1 << 40  # written nowhere
    want_k, want_v = k_cache.clone(), v_cache.clone()
    plain_q, plain_k = rotary(q, k, positions, table)
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < k_cache.shape[0] * block:
            want_k[s // block, :, s % block], want_v[s // block, :, s % block] = plain_k[t], v[t]
    k_out = torch.empty_like(k) if keep else None
    got = rotary_to_cache(q, k, v, positions, table, k_cache, v_cache, slots, k_out=k_out)
    assert torch.equal(got, plain_q) and torch.equal(k_cache, want_k) and torch.equal(v_cache, want_v)
    assert not keep or torch.equal(k_out, plain_k)
    # slots outside heads
    loose = [torch.zeros_like(t).transpose(1, 2).contiguous().transpose(1, 2) for t in (k_cache, v_cache)]
    rotary_to_cache(q, k, v, positions, table, *loose, slots)
    written = [s for s in slots.tolist() if 0 <= s < k_cache.shape[0] * block]
    for s in written:
        assert torch.equal(loose[0][s // block, :, s % block], want_k[s // block, :, s % block])
        assert torch.equal(loose[1][s // block, :, s % block], want_v[s // block, :, s % block])


def test_positions_outside_the_table_are_nan(device):
    q, k, _, _ = inputs(4, 2, 1, 64, torch.float16, device)
    table = rotary_table(10, 32, device=device)
    positions = torch.tensor([-1, 10, 2 ** 31 - 1, 9], dtype=torch.int32, device=device)
    got = rotary(q, k, positions, table)[0]
    assert got[:3, :, :32].isnan().all() and torch.equal(got[:3, :, 32:], q[:3, :, 32:])
    check(got[3:], q[3:], positions[3:], table, False)


def test_long_positions_keep_their_angles(device):
    """An angle of position 2^20 is the 64-bit one, not fp32 position times frequency."""
    table = rotary_table(2 ** 20 + 1, 64, device=device)
    at = torch.arange(0, 64, 2, dtype=torch.float64) / 64
    angle = 2 ** 20 * 10000.0 ** -at
    want = torch.cat([angle.cos(), angle.sin()])
    assert (table[-1].cpu().double() - want).abs().max() <= 2.0 ** -24 + 2 ** 20 * 2.0 ** -51


def test_cache_offsets_past_32_bits(device):
    block, dim = 16, 128
    pages = 2 ** 32 // (block * dim) + 3
    big = torch.empty(pages, 1, block, dim, device=device, dtype=torch.float16)
    q, k, v, positions = inputs(5, 1, 1, dim, torch.float16, device)
    table = rotary_table(5000, dim, device=device)
    slots = pages * block - 1 - torch.arange(5, device=device)
    k_out = torch.empty_like(k)
    rotary_to_cache(q, k, v, positions, table, big, torch.empty_like(big[:1]).expand_as(big), slots * 0 - 1)
    rotary_to_cache(q, k, v, positions, table, big, big, slots, k_out=k_out)
    tail = big[-1, 0, -5:].flip(0)
    # one cache for both: each slot holds the turned key or the value
    assert ((tail == k_out[:, 0]) | (tail == v[:, 0])).all()


def test_refusals(device):
    q, k, v, positions = inputs(6, 4, 2, 64, torch.float16, device)
    table = rotary_table(5000, 64, device=device)
    caches = [torch.zeros(4, 2, 16, 64, device=device, dtype=torch.float16) for _ in range(2)]
    slots = torch.arange(6, device=device)
    bad = [
        (dict(q=q[0]), "expected q"), (dict(k=k[:5]), "expected q"), (dict(k=k.float()), "dtype mismatch"),
        (dict(positions=positions.long()), "positions must be"), (dict(positions=positions[:5]), "positions must have"),
        (dict(table=table.half()), "table must be"), (dict(table=table[0]), "table must be"),
        (dict(table=rotary_table(9, 66, device=device)), "rotary_dim"), (dict(table=table[:, ::2]), "contiguous"),
        (dict(q=q.transpose(1, 2).contiguous().transpose(1, 2)), "contiguous last"), (dict(q_out=q[:5]), "q_out must"),
        (dict(q_out=q.float()), "dtype mismatch"), (dict(k_out=k[:, :1]), "k_out must"),
    ]
    for change, message in bad:
        with pytest.raises(ValueError, match=message):
            rotary(**(dict(q=q, k=k, positions=positions, table=table) | change))
    bad = [
        (dict(v=v[:5]), "v must have"), (dict(v=v.float()), "dtype mismatch"), (dict(k_cache=caches[0][0]), "caches"),
        (dict(k_cache=caches[0][:2]), "caches"), (dict(slots=slots.int()), "slots must be"),
        (dict(slots=slots[:5]), "slots must have"), (dict(k_cache=caches[0].float()), "dtype mismatch"),
    ]
    args = dict(q=q, k=k, v=v, positions=positions, table=table, k_cache=caches[0], v_cache=caches[1], slots=slots)
    for change, message in bad:
        with pytest.raises(ValueError, match=message):
            rotary_to_cache(**(args | change))

"""Head norms with rotary positions, their cache write and their gradient, against 64 bits.

Forward: the sum of squares of a head has at most 16 terms in sequence and 5
sums across lanes, so its relative error is below 24 e with e = 2^-24, and that
of r = 1 / s below 12 e + 4 e (a reciprocal root within two units) = 16 e.
x r w and the turn add four roundings: an element is off by at most 24 e times
the sizes of its two products, and half a unit of its type.

Backward: g is off by 2 e of its products, the sum along x by 24 e of its terms,
r enters three times (48 e) and a handful of products follow: 96 e of the sum of
the sizes of all terms. A weight's gradient adds at most as many terms in
sequence as there are heads and tokens, and 64 more across groups and blocks.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from kernelo_b200.kernels.rotary import (norm_rotary, norm_rotary_backward, norm_rotary_to_cache, rotary_table)

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
LEAST = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133, torch.float32: 2.0 ** -140}
DTYPES = tuple(UNIT)
EPS = 1e-6


def pairs(rot, interleaved):
    return (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))


def turned(x, positions, table, interleaved, inverse=False):
    """R x in 64 bits and the sizes of each element's products."""
    rot = table.shape[1]
    row = table.double()[positions.long()][:, None]
    cos, sin = row[..., :rot // 2], row[..., rot // 2:] * (-1 if inverse else 1)
    a, b = pairs(rot, interleaved)
    y, size = x.clone(), x.abs()
    y[..., a], y[..., b] = x[..., a] * cos - x[..., b] * sin, x[..., a] * sin + x[..., b] * cos
    size[..., a], size[..., b] = (x[..., a].abs() * cos.abs() + x[..., b].abs() * sin.abs(),
                                  x[..., a].abs() * sin.abs() + x[..., b].abs() * cos.abs())
    return y, size


def forward(x, w, positions, table, interleaved, eps=EPS):
    xd = x.double()
    u = xd / (xd.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    return turned(u, positions, table, interleaved)


def check(got, x, w, positions, table, interleaved, eps=EPS):
    want, size = forward(x, w, positions, table, interleaved, eps)
    off = 24 * E * size
    assert got.dtype == x.dtype and got.shape == x.shape
    assert ((got.double() - want).abs() <= off + UNIT[x.dtype] * (want.abs() + off) + LEAST[x.dtype]).all()


def check_gradient(got, got_w, dy, x, w, positions, table, interleaved, eps=EPS):
    dim, xd, wd = x.shape[2], x.double(), w.double()
    g, size = turned(dy.double(), positions, table, interleaved, True)
    r = (xd.square().mean(-1, keepdim=True) + eps).rsqrt()
    u = xd * r
    want = r * (g * wd - u * (g * wd * u).mean(-1, keepdim=True))
    off = 96 * E * r * (size * wd.abs() + u.abs() * (size * wd.abs() * u.abs()).mean(-1, keepdim=True))
    assert got.dtype == x.dtype and got.shape == x.shape
    assert ((got.double() - want).abs() <= off + UNIT[x.dtype] * (want.abs() + off) + LEAST[x.dtype]).all()
    want_w, size_w = (g * u).sum((0, 1)), (size * u.abs()).sum((0, 1))
    assert got_w.dtype == torch.float32 and got_w.shape == (dim,)
    assert ((got_w.double() - want_w).abs() <= (x.shape[0] * x.shape[1] + 96) * E * size_w + 2.0 ** -140).all()


def inputs(tokens, heads, kv_heads, dim, dtype, device, most=5000, seed=0):
    gen = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(tokens, h, dim, generator=gen).mul_(torch.rand(tokens, h, 1, generator=gen) * 3 + 0.1).to(dtype).to(device)
               for h in (heads, kv_heads, kv_heads))
    qw, kw = (torch.randn(dim, generator=gen).mul_(0.3).add_(1.0).to(dtype).to(device) for _ in range(2))
    return q, k, v, qw, kw, torch.randint(0, most, (tokens,), generator=gen, dtype=torch.int32).to(device)


def both(q, k, qw, kw, positions, table, interleaved):
    for x, w, y in zip((q, k), (qw, kw), norm_rotary(q, k, positions, table, qw, kw, eps=EPS, interleaved=interleaved)):
        check(y, x, w, positions, table, interleaved)
    gen = torch.Generator().manual_seed(7)
    dq, dk = (torch.randn(x.shape, generator=gen).to(x.dtype).to(x.device) for x in (q, k))
    gq, gk, gqw, gkw = norm_rotary_backward(dq, dk, q, k, positions, table, qw, kw, eps=EPS, interleaved=interleaved)
    check_gradient(gq, gqw, dq, q, qw, positions, table, interleaved)
    check_gradient(gk, gkw, dk, k, kw, positions, table, interleaved)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rot", [(128, 128), (128, 64), (64, 64), (80, 80), (80, 40), (80, 20), (96, 24), (20, 6),
                                     (36, 32), (7, 4), (256, 256), (256, 0), (64, 2), (2, 2), (1, 0), (250, 250),
                                     (255, 100), (236, 236), (32, 32)])
def test_layouts_and_parts(dim, rot, interleaved, dtype, device):
    q, k, _, qw, kw, positions = inputs(37, 5, 3, dim, dtype, device)
    table = rotary_table(5000, rot, device=device) if rot else torch.empty(5000, 0, device=device)
    both(q, k, qw, kw, positions, table, interleaved)


@pytest.mark.parametrize("tokens,heads,kv_heads", [(1, 1, 1), (1, 32, 8), (3, 7, 1), (1000, 8, 8), (2049, 4, 2), (5, 70, 70),
                                                   (9, 3, 0), (9, 0, 3)])
def test_sizes(tokens, heads, kv_heads, device):
    q, k, _, qw, kw, positions = inputs(tokens, heads, kv_heads, 128, torch.bfloat16, device)
    both(q, k, qw, kw, positions, rotary_table(5000, 128, device=device), False)


def test_no_tokens(device):
    q, k, _, qw, kw, positions = inputs(3, 4, 2, 64, torch.float16, device)
    table = rotary_table(50, 64, device=device)
    for x in norm_rotary(q[:0], k[:0], positions[:0], table, qw, kw):
        assert x.shape[0] == 0
    gq, gk, gqw, gkw = norm_rotary_backward(q[:0], k[:0], q[:0], k[:0], positions[:0], table, qw, kw)
    assert gq.shape == (0, 4, 64) and gk.shape == (0, 2, 64)
    assert torch.equal(gqw, torch.zeros_like(gqw)) and torch.equal(gkw, torch.zeros_like(gkw))


@pytest.mark.parametrize("dtype", DTYPES)
def test_views_in_place_and_odd_strides(dtype, device):
    qkv = torch.randn(65, 12, 64, device=device).to(dtype)
    _, _, _, qw, kw, _ = inputs(1, 1, 1, 64, dtype, device)
    positions = torch.arange(65, dtype=torch.int32, device=device)
    table = rotary_table(65, 32, device=device)
    q, k = qkv[:, :8], qkv[:, 8:10]
    before, rest = qkv.clone(), qkv[:, 10:].clone()
    a, b = norm_rotary(q, k, positions, table, qw, kw, eps=EPS)
    got = norm_rotary(q, k, positions, table, qw, kw, eps=EPS, q_out=q, k_out=k)
    assert got[0] is q and torch.equal(q, a) and torch.equal(k, b) and torch.equal(qkv[:, 10:], rest)
    check(q, before[:, :8], qw, positions, table, False)
    odd = torch.randn(65, 5, 67, device=device).to(dtype)
    weights = torch.randn(2, 67, device=device).to(dtype)
    for interleaved in (False, True):
        both(odd[:, :4, 1:65], odd[:, 4:, 3:67], weights[0, 1:65], weights[1, 2:66], positions, table, interleaved)
    # gradients that are broadcast, as a sum's or a mean's are
    dq, dk = (torch.full((1, 1, 64), 0.25, device=device, dtype=dtype).expand(65, n, 64) for n in (8, 2))
    gq, gk, gqw, gkw = norm_rotary_backward(dq, dk, before[:, :8], before[:, 8:10], positions, table, qw, kw, eps=EPS)
    check_gradient(gq, gqw, dq, before[:, :8], qw, positions, table, False)
    check_gradient(gk, gkw, dk, before[:, 8:10], kw, positions, table, False)


@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient_against_differences(interleaved, device):
    """Central differences of <dy, y(x, w)> in 64 bits, step 2^-14: off by a third derivative (below 2^6 for these
    sizes) times 2^-28 / 6, and by the rounding of values below 2^8 at 2^-52 2^14."""
    q, k, _, qw, kw, positions = inputs(5, 3, 2, 16, torch.float32, device)
    q, k = (x / x.square().mean(-1, keepdim=True).sqrt() for x in (q, k))
    table = rotary_table(5000, 12, device=device)
    dq, dk = torch.randn_like(q), torch.randn_like(k)
    got = norm_rotary_backward(dq, dk, q, k, positions, table, qw, kw, eps=EPS, interleaved=interleaved)
    step = 2.0 ** -14
    for x, w, dy, gx, gw in ((q, qw, dq, got[0], got[2]), (k, kw, dk, got[1], got[3])):
        x, w = x.double(), w.double()

        def value(x, w):
            return (forward(x, w, positions, table, interleaved)[0] * dy.double())

        for e in range(16):
            d = torch.zeros(16, dtype=torch.float64, device=device)
            d[e] = step
            slope = (value(x + d, w) - value(x - d, w)).sum(-1) / (2 * step)
            assert ((gx[..., e].double() - slope).abs() <= 2.0 ** -18).all()
            slope = (value(x, w + d) - value(x, w - d)).sum() / (2 * step)
            assert (gw[e].double() - slope).abs() <= 2.0 ** -16


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,rot,block", [(128, 128, 16), (64, 32, 24), (20, 6, 5)])
@pytest.mark.parametrize("keep", [False, True])
def test_cache_write(dim, rot, block, keep, dtype, device):
    q, k, v, qw, kw, positions = inputs(50, 6, 2, dim, dtype, device)
    table = rotary_table(5000, rot, device=device)
    k_cache = torch.full((9 + 50 // block, 2, block, dim), 5.0, device=device, dtype=dtype)
    v_cache = torch.full_like(k_cache, 6.0)
    places = np.random.default_rng(0).permutation(k_cache.shape[0] * block)[:50]
    slots = torch.from_numpy(places).to(device)
    slots[3], slots[7], slots[9] = -1, k_cache.shape[0] * block, 1 << 40  # written nowhere
    want_k, want_v = k_cache.clone(), v_cache.clone()
    plain_q, plain_k = norm_rotary(q, k, positions, table, qw, kw, eps=EPS)
    for t, slot in enumerate(slots.tolist()):
        if 0 <= slot < k_cache.shape[0] * block:
            want_k[slot // block, :, slot % block] = plain_k[t]
            want_v[slot // block, :, slot % block] = v[t]
    k_out = torch.empty_like(k) if keep else None
    got = norm_rotary_to_cache(q, k, v, positions, table, qw, kw, k_cache, v_cache, slots, eps=EPS, k_out=k_out)
    assert torch.equal(got, plain_q) and torch.equal(k_cache, want_k) and torch.equal(v_cache, want_v)
    assert k_out is None or torch.equal(k_out, plain_k)


def test_caches_of_other_orders(device):
    """Pages stored slot by slot, and a cache whose pages lie far apart."""
    q, k, v, qw, kw, positions = inputs(40, 6, 2, 64, torch.bfloat16, device)
    table = rotary_table(5000, 64, device=device)
    _, plain_k = norm_rotary(q, k, positions, table, qw, kw)
    slots = torch.randperm(80, device=device)[:40]
    for make in (lambda: torch.zeros(5, 16, 2, 64, device=device, dtype=torch.bfloat16).transpose(1, 2),
                 lambda: torch.zeros(10, 3, 19, 72, device=device, dtype=torch.bfloat16)[::2, 1:, 2:18, 8:]):
        k_cache, v_cache = make(), make()
        norm_rotary_to_cache(q, k, v, positions, table, qw, kw, k_cache, v_cache, slots)
        assert torch.equal(k_cache[slots // 16, :, slots % 16], plain_k)
        assert torch.equal(v_cache[slots // 16, :, slots % 16], v)
        assert torch.count_nonzero(k_cache) <= 40 * 2 * 64


@pytest.mark.parametrize("dtype", DTYPES)
def test_positions_outside_the_table_and_extreme_heads(dtype, device):
    q, k, _, qw, kw, positions = inputs(12, 4, 2, 64, dtype, device)
    table = rotary_table(100, 32, device=device)
    positions = torch.arange(12, dtype=torch.int32, device=device)
    positions[4], positions[5], positions[6] = -1, 100, 2 ** 31 - 1
    q[0], q[1, 2] = 0.0, torch.finfo(dtype).max if dtype != torch.float32 else 1e15
    q[2, 1, 7], q[3, 1, 7] = torch.inf, torch.nan
    y, _ = norm_rotary(q, k, positions, table, qw, kw, eps=EPS)
    assert torch.isnan(y[4:7, :, :32]).all() and torch.isfinite(y[4:7, :, 32:]).all()
    assert torch.equal(y[0], torch.zeros_like(y[0]))  # a head of zeros stays zeros
    plain = torch.ones(12, 4, dtype=torch.bool, device=device)
    plain[4:7], plain[2:4, 1] = False, False
    assert torch.isfinite(y[plain]).all()
    assert torch.isnan(y[3, 1]).all() and not torch.isfinite(y[2, 1, 7])
    near = positions.clamp(0, 99)
    want, size = forward(q, qw, near, table, False)
    off = 24 * E * size
    assert ((y.double() - want).abs() <= off + UNIT[dtype] * (want.abs() + off) + LEAST[dtype])[plain].all()
    # the least number whose square is lost in fp32 is as nothing beside eps
    tiny = torch.full_like(q, 2.0 ** -24)
    check(norm_rotary(tiny, k, near, table, qw, kw, eps=EPS)[0], tiny, qw, near, table, False)
    gq, _, gqw, _ = norm_rotary_backward(torch.ones_like(q), torch.ones_like(k), q, k, positions, table, qw, kw, eps=EPS)
    assert torch.isfinite(gq[7:]).all() and torch.isnan(gq[4:7, :, :32]).all() and torch.isnan(gqw[:32]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_heads_whose_squares_fp32_cannot_hold(dtype, device):
    q, k, _, qw, kw, positions = inputs(7, 4, 2, 64, dtype, device)
    table = rotary_table(5000, 64, device=device)
    most = torch.finfo(dtype).max
    both((q / q.abs().max()).mul(most).to(dtype), (k.sign() * most).to(dtype), qw, kw, positions, table, False)


def test_captured_replayed_and_on_another_stream(device):
    """A graph replayed with other operands, beside eager calls; forward and backward; the same bits each time."""
    shape = (300, 8, 2, 128)
    q, k, v, qw, kw, positions = inputs(*shape, torch.bfloat16, device)
    table = rotary_table(5000, 128, device=device)
    caches = [torch.zeros(30, 2, 16, 128, device=device, dtype=torch.bfloat16) for _ in range(2)]
    slots = torch.randperm(480, device=device)[:300]
    dq, dk = torch.randn_like(q), torch.randn_like(k)

    def step():
        out = norm_rotary_to_cache(q, k, v, positions, table, qw, kw, *caches, slots)
        return out, *norm_rotary_backward(dq, dk, q, k, positions, table, qw, kw)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (1, 2):
        for to, new in zip((q, k, v, qw, kw, positions), inputs(*shape, torch.bfloat16, device, seed=seed)):
            to.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        held, kept = [x.clone() for x in captured], [c.clone() for c in caches]
        with torch.cuda.stream(side):
            eager = step()
        side.synchronize()
        for a, b in zip(held + kept, [*eager, *caches]):
            assert torch.equal(a, b)
        check(held[0], q, qw, positions, table, False, 1e-5)


def test_refusals(device):
    q, k, v, qw, kw, positions = inputs(6, 4, 2, 64, torch.float16, device)
    table = rotary_table(50, 64, device=device)
    cache = torch.zeros(3, 2, 16, 64, device=device, dtype=torch.float16)
    slots = torch.arange(6, device=device)
    for change, message in ((dict(q_weight=qw[:32]), "q_weight must have shape"), (dict(k_weight=kw.float()), "dtype mismatch"),
                            (dict(k_weight=kw.cpu()), "one device"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
                            (dict(q_weight=torch.zeros(128, device=device).half()[::2]), "contiguous"),
                            (dict(q_out=k), "q_out must have shape"), (dict(positions=positions.long()), "positions"),
                            (dict(q_out=torch.zeros_like(q).float()), "dtype mismatch"),
                            (dict(table=table[:, :63]), "table")):
        operands = dict(q=q, k=k, positions=positions, table=table, q_weight=qw, k_weight=kw) | change
        with pytest.raises(ValueError, match=message):
            norm_rotary(**operands)
    wide = torch.zeros(2, 1, 258, device=device)
    with pytest.raises(ValueError, match="at most 256"):
        norm_rotary(wide, wide, positions[:2], table, wide[0, 0], wide[0, 0])
    buf = torch.zeros(6, 9, 64, device=device, dtype=torch.float16)
    for q_out, k_out, message in ((buf[:, 1:5], buf[:, 5:7], "q_out shares memory with q"),
                                  (buf[:, 4:8], None, "q_out shares memory with k"),
                                  (None, buf[:, 2:4], "k_out shares memory with q"),
                                  (buf[:, :4], buf[:, 3:5], "k_out shares memory")):
        with pytest.raises(ValueError, match=message):
            norm_rotary(buf[:, :4], buf[:, 5:7], positions, table, qw, kw, q_out=q_out, k_out=k_out)
    with pytest.raises(ValueError, match="q_out shares memory with v"):
        norm_rotary_to_cache(q, buf[:, 2:4], buf[:, 6:8], positions, table, qw, kw, cache, cache.clone(), slots,
                             q_out=buf[:, 5:9])
    with pytest.raises(ValueError, match="slots"):
        norm_rotary_to_cache(q, k, v, positions, table, qw, kw, cache, cache.clone(), slots.int())
    with pytest.raises(ValueError, match="dq must have shape"):
        norm_rotary_backward(k, k, q, k, positions, table, qw, kw)
    with pytest.raises(ValueError, match="dtype mismatch"):
        norm_rotary_backward(q.float(), k, q, k, positions, table, qw, kw)

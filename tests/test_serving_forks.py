"""A server that answers prompts several ways from one cache: requests fork, go on apart, are penalised and masked, end,
and their pages are moved together; against whole sequences in plain PyTorch fp64.

Outputs are held to the gate's threshold of their type (``kernelo_b200.testing``), as those of the block are elsewhere.
"""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

from kernelo_b200.integration import PagedCache, ServingBlock, ServingConfig, ServingHead
from kernelo_b200.integration.serving import Step
from kernelo_b200.testing import assert_verified

TINY = ServingConfig(hidden=256, heads=8, kv_heads=2, intermediate=512, block_size=8, max_positions=512, qk_norm=True)
VOCAB = 501


def plain_block(block, x):
    """One causal sequence (tokens, hidden)."""
    c, dim, n = block.config, block.config.head_dim, x.shape[0]
    w = {name: p.detach().double() for name, p in block.named_parameters()}
    x = x.double()

    def norm(h, gamma):
        return h * torch.rsqrt(h.square().mean(-1, keepdim=True) + c.eps) * gamma

    qkv = (norm(x, w["attn_norm_weight"]) @ w["qkv_proj.weight"].T).view(n, c.heads + 2 * c.kv_heads, dim)
    at = torch.arange(n, device=x.device)
    angle = at.double()[:, None] * c.rotary_base ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=x.device) / dim)
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]

    def rotate(t):
        z = torch.complex(t[..., :dim // 2], t[..., dim // 2:]) * turn
        return torch.cat([z.real, z.imag], -1)

    q, k, v = qkv.split([c.heads, c.kv_heads, c.kv_heads], 1)
    if c.qk_norm:
        q, k = norm(q, w["q_norm_weight"]), norm(k, w["k_norm_weight"])
    q, k = rotate(q), rotate(k)
    k, v = (t.repeat_interleave(c.heads // c.kv_heads, 1) for t in (k, v))
    scores = torch.einsum("ihd,jhd->hij", q, k) * dim ** -0.5
    weights = scores.masked_fill(at[None, :] > at[:, None], -torch.inf).softmax(-1)
    x = x + torch.einsum("hij,jhd->ihd", weights, v).reshape(x.shape) @ w["out_proj.weight"].T
    up = F.gelu(norm(x, w["mlp_norm_weight"]) @ w["mlp_up.weight"].T + w["mlp_up.bias"], approximate="tanh")
    return x + up @ w["mlp_down.weight"].T


def make(cls, *args, dtype, device):
    torch.manual_seed(0)
    module = cls(*args, dtype=dtype, device=device)
    with torch.no_grad():
        for name, p in module.named_parameters():
            p.normal_(0.0, 0.06)
            if "norm_weight" in name:
                p.add_(1.0)
    return module


def test_forks_and_releases_that_are_refused_on_the_host():
    cache = PagedCache(TINY, requests=5, blocks=6, device="cpu")
    cache.lens, cache.free = [20, 9, 3, 0, 0], cache.free[:0]
    before = cache.block_table.clone()
    for parents, children, message in (([0], [5], "request must be"), ([-1], [3], "request must be"), ([0, 1], [3, 3], "of its own"),
                                       ([0, 3], [3, 4], "of its own"), ([0], [3, 4], "of its own"), ([0], [2], "have tokens"),
                                       ([0, 1], [3, 4], "2 pages too few")):
        with pytest.raises(ValueError, match=message):
            cache.fork(parents, children)
    with pytest.raises(ValueError, match="request must be"):
        cache.release([0, 7])
    assert cache.lens == [20, 9, 3, 0, 0] and torch.equal(cache.block_table, before)
    assert cache._together == [[]] * 5


def test_several_requests_released_at_once_on_the_host():
    cache = PagedCache(TINY, requests=3, blocks=9, device="cpu")
    cache.lens, cache.free = [17, 8, 1], cache.free[5:]
    cache.block_table[0, :3], cache.block_table[1, 0], cache.block_table[2, 0] = torch.tensor([4, 0, 3], dtype=torch.int32), 2, 1
    cache.release([2, 0, 2])
    assert cache.lens == [0, 8, 0] and cache.free.tolist() == [5, 6, 7, 8, 1, 4, 0, 3]
    assert (cache.block_table[[0, 2]] == -1).all() and cache.block_table[1, 0] == 2


def test_a_step_planned_before_the_pages_moved_is_refused():
    cache = PagedCache(TINY, requests=2, blocks=9, device="cpu")
    step = Step((1, 1), None, None, (0, 0), moved=0)
    cache.check_step(step)
    cache.check_step(Step((1, 1), None, None))
    cache._moved = 1
    with pytest.raises(ValueError, match="before the cache's pages moved"):
        cache.advance(step)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_prompts_forked_continued_released_and_moved(dtype, device):
    block = make(ServingBlock, TINY, dtype=dtype, device=device)
    head = make(ServingHead, TINY, VOCAB, dtype=dtype, device=device)
    cache = PagedCache(TINY, requests=7, blocks=40, dtype=dtype, device=device)
    cache.k.fill_(torch.nan)  # pages start as anything
    cache.v.fill_(torch.nan)
    gen = torch.Generator(device=device).manual_seed(1)
    empty = torch.empty(0, TINY.hidden, device=device, dtype=dtype)
    history = [empty] * 7

    def go(new, call):
        parts, step = [torch.randn(n, TINY.hidden, generator=gen, device=device).to(dtype) for n in new], cache.plan(new)
        got = call(torch.cat(parts), cache, step)
        cache.advance(step)
        want = []
        for r, x in enumerate(parts):
            history[r] = torch.cat([history[r], x])
            if x.shape[0]:
                want.append(plain_block(block, history[r])[-x.shape[0]:])
        assert_verified(torch.cat(want), got, dtype=dtype, context=f"tokens {new}")
        return got

    def fork(parents, children):
        cache.fork(parents, children)
        for p, c in zip(parents, children):
            history[c] = history[p]

    def release(*requests):
        cache.release(list(requests))
        for r in requests:
            history[r] = empty

    def pages():
        """Every page is free or held, and held as often as the counts say."""
        held = [p for r, n in enumerate(cache.lens) for p in cache.block_table[r, :-(-n // 8)].tolist()]
        assert sorted(set(held) | set(cache.free.tolist())) == list(range(40)) and not set(held) & set(cache.free.tolist())
        assert len(set(cache.free.tolist())) == cache.free.shape[0]
        assert cache.holders.tolist() == [max(held.count(p) - 1, 0) for p in range(40)]
        assert cache.lens == [h.shape[0] for h in history]
        return held

    with torch.inference_mode():
        go((21, 16, 0, 0, 0, 0, 0), block.prompts)
        fork([0, 0, 1], [2, 3, 4])
        held = pages()
        assert len(held) == 3 + 2 + 3 + 3 + 2 and len(set(held)) == 3 + 2 + 1 + 1
        go((1, 1, 1, 1, 1, 0, 0), block.tokens)
        go((3, 0, 9, 1, 2, 0, 0), block.tokens)
        fork([2, 3, ], [5, 6])  # forks of forks
        pages()
        go((1, 1, 1, 1, 1, 1, 1), block.tokens)
        release(0, 5)
        pages()
        go((0, 1, 1, 2, 1, 0, 12), block.tokens)
        stale = cache.plan((0, 1, 1, 1, 1, 0, 1))
        live = cache.compact()
        assert sorted(set(pages())) == list(range(live)) and cache.free.tolist() == list(range(live, 40))
        with pytest.raises(ValueError, match="before the cache's pages moved"):
            block.tokens(torch.zeros(5, TINY.hidden, device=device, dtype=dtype), cache, stale)
        last = go((0, 1, 1, 1, 1, 0, 1), block.tokens)

        # their next tokens: a history each, one that has a bias, one under a grammar
        tokens = torch.randint(0, VOCAB, (5, 30), generator=gen, device=device, dtype=torch.int32)
        lens = torch.tensor([30, 0, 7, 12, 1], dtype=torch.int32, device=device)
        penalty = torch.tensor([1.3, 1.0, 1.1, 2.0, 1.2], device=device)
        bias_tokens = torch.tensor([[-1], [5], [-1], [-1], [-1]], dtype=torch.int32, device=device)
        bias = torch.full((5, 1), 3.0, device=device)
        allowed = torch.zeros(1, -(-VOCAB // 32), dtype=torch.int32, device=device)
        allowed[0, 0], allowed[0, 15] = 0b1011, 1 << 20
        which = torch.tensor([-1, -1, 0, -1, -1], dtype=torch.int32, device=device)
        asked = dict(tokens=tokens, token_lens=lens, repetition=penalty, presence=penalty, bias_tokens=bias_tokens,
                     bias_values=bias, allowed=allowed, allowed_rows=which)
        p = head(last, **asked)
        x = last.double()
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + TINY.eps) * head.norm_weight.double()
        logits = x @ head.vocab_proj.weight.double().T
        assert_verified(logits.softmax(-1), head(last), dtype=dtype, context="head")
        for r in range(5):
            seen = tokens[r, :lens[r]].long().unique()
            y = logits[r, seen]
            logits[r, seen] = torch.where(y > 0, y / penalty[r], y * penalty[r]) - penalty[r]
        logits[1, 5] += 3.0
        off = torch.ones(VOCAB, dtype=torch.bool, device=device)
        off[[0, 1, 3, 500]] = False
        logits[2, off] = -torch.inf
        assert_verified(logits.softmax(-1), p, dtype=dtype, context="adjusted head")
        assert not p[2, off].any()

        release(1, 2, 3, 4, 6)
        assert pages() == [] and cache.compact() == 0


@pytest.mark.gpu
def test_forks_until_the_pool_is_full(device):
    cache = PagedCache(TINY, requests=8, blocks=6, device=device)
    cache.advance(cache.plan((20,) + (0,) * 7))  # three pages, the last one partial
    cache.fork([0, 0, 0], [1, 2, 3])
    assert cache.free.shape[0] == 0
    with pytest.raises(ValueError, match="1 pages too few"):
        cache.fork([0], [4])
    cache.release(2)
    cache.fork([0], [4])
    cache.release([0, 1, 3])
    assert cache.free.shape[0] == 3 and cache.holders.tolist() == [0] * 6
    cache.release(4)
    assert sorted(cache.free.tolist()) == list(range(6))

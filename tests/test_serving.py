"""A decoder block served from a paged cache, against the same block in plain PyTorch fp64 on whole sequences.

The block's kernels are the ones checked alone elsewhere; here the plan, the
pages, the rotary positions and the attention have to fit together. Outputs are
held to the gate's threshold of their type (``kernelo_b200.testing``): several
16-bit roundings lie between input and output.
"""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

from kernelo_b200.integration import PagedCache, ServingBlock, ServingConfig
from kernelo_b200.testing import assert_verified

TINY = ServingConfig(hidden=256, heads=8, kv_heads=2, intermediate=512, block_size=8, max_positions=512)


def test_configuration_is_checked():
    assert TINY.head_dim == 32
    with pytest.raises(ValueError, match="key heads"):
        ServingConfig(hidden=256, heads=8, kv_heads=3, intermediate=512)
    with pytest.raises(ValueError, match="not divisible"):
        ServingConfig(hidden=250, heads=8, kv_heads=2, intermediate=512)
    with pytest.raises(ValueError, match="block_size"):
        ServingConfig(hidden=256, heads=8, kv_heads=2, intermediate=512, block_size=0)


def test_plans_the_cache_cannot_hold_are_refused_on_the_host():
    cache = PagedCache(TINY, requests=2, blocks=5, device="cpu")
    for lens, message in (([1], "2 token counts"), ([1, -1], "token counts"), ([513, 0], "512 positions"),
                          ([33, 8], "1 pages too few")):
        with pytest.raises(ValueError, match=message):
            cache.plan(lens)


def plain_block(block: ServingBlock, x: torch.Tensor, positions: torch.Tensor, seen: torch.Tensor) -> torch.Tensor:
    """One sequence (tokens, hidden) in fp64; ``seen`` (tokens, tokens): what attends to what."""
    c, dim = block.config, block.config.head_dim
    w = {n: p.detach().double() for n, p in block.named_parameters()}
    x = x.double()

    def norm(h, gamma):
        return h * torch.rsqrt(h.square().mean(-1, keepdim=True) + c.eps) * gamma

    qkv = (norm(x, w["attn_norm_weight"]) @ w["qkv_proj.weight"].T).view(x.shape[0], c.heads + 2 * c.kv_heads, dim)
    angle = positions.double()[:, None] * c.rotary_base ** (
        -torch.arange(0, dim, 2, dtype=torch.float64, device=x.device) / dim)
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]

    def rotate(t):
        z = torch.complex(t[..., :dim // 2], t[..., dim // 2:]) * turn
        return torch.cat([z.real, z.imag], -1)

    q, k, v = qkv.split([c.heads, c.kv_heads, c.kv_heads], 1)
    q, k = rotate(q), rotate(k)
    k, v = (t.repeat_interleave(c.heads // c.kv_heads, 1) for t in (k, v))
    scores = torch.einsum("ihd,jhd->hij", q, k) * dim ** -0.5
    weights = scores.masked_fill(~seen, -torch.inf).softmax(-1)
    x = x + torch.einsum("hij,jhd->ihd", weights, v).reshape(x.shape) @ w["out_proj.weight"].T
    up = F.gelu(norm(x, w["mlp_norm_weight"]) @ w["mlp_up.weight"].T + w["mlp_up.bias"], approximate="tanh")
    return x + up @ w["mlp_down.weight"].T


def make_block(dtype, device):
    torch.manual_seed(0)
    block = ServingBlock(TINY, dtype=dtype, device=device)
    with torch.no_grad():
        for p in block.parameters():
            p.normal_(0.0, 0.06)
        block.attn_norm_weight.add_(1.0)
        block.mlp_norm_weight.add_(1.0)
    return block


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_prompts_then_tokens_then_trees(dtype, device):
    block = make_block(dtype, device)
    cache = PagedCache(TINY, requests=3, blocks=80, dtype=dtype, device=device)
    cache.k.fill_(torch.nan)  # pages start as anything
    cache.v.fill_(torch.nan)
    gen = torch.Generator(device=device).manual_seed(1)
    history = [torch.empty(0, TINY.hidden, device=device, dtype=dtype) for _ in range(3)]

    def fresh(lens):
        return [torch.randn(n, TINY.hidden, generator=gen, device=device).to(dtype) for n in lens]

    def expect(r, extra, positions=None, seen=None):
        x = torch.cat([history[r], extra])
        n, m = x.shape[0], extra.shape[0]
        positions = torch.arange(n, device=device) if positions is None else positions
        full = torch.ones(n, n, dtype=torch.bool, device=device).tril()
        if seen is not None:
            full[n - m:, n - m:] = seen
        return plain_block(block, x, positions, full)[n - m:]

    with torch.inference_mode():
        # prompts of different lengths, one request not started yet
        parts, step = fresh((70, 0, 21)), cache.plan((70, 0, 21))
        got = block.prompts(torch.cat(parts), cache, step)
        assert_verified(torch.cat([expect(r, parts[r]) for r in range(3)]), got, dtype=dtype, context="prompts")
        cache.advance(step)
        history = [torch.cat([h, x]) for h, x in zip(history, parts)]
        # one token each; the second request's first
        for _ in range(3):
            parts, step = fresh((1, 1, 1)), cache.plan((1, 1, 1))
            got = block.tokens(torch.cat(parts), cache, step)
            assert_verified(torch.cat([expect(r, parts[r]) for r in range(3)]), got, dtype=dtype, context="tokens")
            cache.advance(step)
            history = [torch.cat([h, x]) for h, x in zip(history, parts)]
        # drafts as trees: node 1 and 2 follow 0, node 3 follows 1
        parts, step = fresh((4, 4, 4)), cache.plan((4, 4, 4))
        seen = torch.tensor([[1, 0, 0, 0], [1, 1, 0, 0], [1, 0, 1, 0], [1, 1, 0, 1]], dtype=torch.bool, device=device)
        words = torch.tensor([[0b0001], [0b0011], [0b0101], [0b1011]] * 3, device=device)
        depths = torch.tensor([0, 1, 1, 2] * 3, dtype=torch.int32, device=device)
        got = block.tokens(torch.cat(parts), cache, step, words, depths)
        want = []
        for r in range(3):
            n = history[r].shape[0]
            positions = torch.cat([torch.arange(n, device=device), n + depths[:4].long()])
            want.append(expect(r, parts[r], positions, seen))
        assert_verified(torch.cat(want), got, dtype=dtype, context="trees")
        # the first two nodes are kept of the first request, none of the others': their pages go back
        taken = cache.free.shape[0]
        cache.advance(step, kept=(2, 0, 0))
        assert cache.lens == [75, 3, 24] and cache.free.shape[0] >= taken - 3
        history[0] = torch.cat([history[0], parts[0][:2]])
        used = sum(-(-n // TINY.block_size) for n in cache.lens)
        assert cache.free.shape[0] == 80 - used and len(set(cache.free.tolist())) == 80 - used
        # and the next tokens, chains of several, go on from what was kept
        parts, step = fresh((3, 9, 1)), cache.plan((3, 9, 1))
        got = block.tokens(torch.cat(parts), cache, step)
        assert_verified(torch.cat([expect(r, parts[r]) for r in range(3)]), got, dtype=dtype, context="after drafts")


@pytest.mark.gpu
def test_malformed_calls_are_refused(device):
    block = make_block(torch.float16, device)
    cache = PagedCache(TINY, requests=1, blocks=8, device=device)
    step = cache.plan([9])
    with pytest.raises(ValueError, match="expected"):
        block.prompts(torch.zeros(9, 128, device=device, dtype=torch.float16), cache, step)
    block.prompts(torch.zeros(9, 256, device=device, dtype=torch.float16), cache, step)
    with pytest.raises(ValueError, match="kept"):
        cache.advance(step, kept=[10])
    cache.advance(step)
    with pytest.raises(ValueError, match="starts requests"):
        block.prompts(torch.zeros(1, 256, device=device, dtype=torch.float16), cache, cache.plan([1]))

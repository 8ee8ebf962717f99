"""A decoder block served from a paged key/value cache, on the native kernels alone.

:class:`~kernelo_b200.integration.transformer.TransformerBlock` runs batches of
equal length and leaves attention to PyTorch. A server has prompts of different
lengths, grouped key heads, rotary positions, and a cache of pages that its
decoding steps -- one token or a tree of drafted ones per request -- extend:

    cache = PagedCache(config, requests=2, blocks=64)
    step = cache.plan([700, 31])              # pages, positions and slots, on the GPU
    y = block.prompts(x, cache, step)         # x: all prompts' tokens, packed
    cache.advance(step)
    step = cache.plan([4, 4])                 # four drafted tokens each ..
    y = block.tokens(x, cache, step, mask, depths)  # ... that see their ancestors
    cache.advance(step, kept=[[0, 1, 3], 1])  # the accepted branch, or the first so many (the rest is written over)
    cache.release(0)                          # finished: its pages go back, its row takes another request
"""

from __future__ import annotations

from dataclasses import dataclass

import torch
from torch import nn

from kernelo_b200.integration.transformer import BlockConfig
from kernelo_b200.kernels.attention import prefill_attention, tree_attention
from kernelo_b200.kernels.fused_linear import fused_linear_gelu
from kernelo_b200.kernels.matmul import matmul
from kernelo_b200.kernels.paged import StepSlots, build_slots
from kernelo_b200.kernels.rmsnorm import rmsnorm
from kernelo_b200.kernels.rotary import rotary_table, rotary_to_cache


@dataclass(frozen=True)
class ServingConfig(BlockConfig):
    """A block's geometry and its cache's: grouped key heads, pages, positions."""

    kv_heads: int = 8
    block_size: int = 16
    max_positions: int = 8192
    rotary_base: float = 10000.0

    def __post_init__(self) -> None:
        super().__post_init__()
        if self.kv_heads < 1 or self.heads % self.kv_heads:
            raise ValueError(f"{self.heads} heads are not a multiple of {self.kv_heads} key heads")
        if self.block_size < 1:
            raise ValueError(f"block_size must be positive, got {self.block_size}")


@dataclass(frozen=True)
class Step:
    """Tokens that a forward pass adds to the cache's requests."""

    new_lens: tuple[int, ...]
    slots: StepSlots
    context_lens: torch.Tensor  # tokens of each request before the step
    lens: tuple[int, ...] | None = None  # the same on the host


class PagedCache:
    """Keys and values of a fixed set of requests in pages ``(blocks, kv_heads, block, dim)``.

    The caller's lengths plan each step; pages move from the free list to the
    block table on the GPU, and nothing is read back.
    """

    def __init__(self, config: ServingConfig, *, requests: int, blocks: int, dtype: torch.dtype = torch.float16,
                 device: torch.device | str = "cuda") -> None:
        shape = (blocks, config.kv_heads, config.block_size, config.head_dim)
        self.config = config
        self.k, self.v = (torch.empty(shape, dtype=dtype, device=device) for _ in range(2))
        per_request = -(-config.max_positions // config.block_size)
        self.block_table = torch.full((requests, per_request), -1, dtype=torch.int32, device=device)
        self.free = torch.arange(blocks, dtype=torch.int32, device=device)
        self.lens = [0] * requests

    def _device_ints(self, values) -> torch.Tensor:
        return torch.tensor(values, dtype=torch.int32).to(self.free.device, non_blocking=True)

    def _pages(self, new_lens) -> list[int]:
        """Pages of each request once it has ``new_lens[r]`` tokens more."""
        return [-(-(n + a) // self.config.block_size) for n, a in zip(self.lens, new_lens)]

    def plan(self, new_lens) -> Step:
        """Pages and slots for ``new_lens[r]`` tokens more of each request."""
        new_lens = tuple(int(n) for n in new_lens)
        if len(new_lens) != len(self.lens) or min(new_lens, default=0) < 0:
            raise ValueError(f"expected {len(self.lens)} token counts, got {new_lens}")
        if any(n + a > self.config.max_positions for n, a in zip(self.lens, new_lens)):
            raise ValueError(f"a request would pass {self.config.max_positions} positions")
        short = sum(self._pages(new_lens)) - sum(self._pages([0] * len(new_lens))) - self.free.shape[0]
        if short > 0:
            raise ValueError(f"the cache has {short} pages too few for this step")
        context = self._device_ints(self.lens)
        slots = build_slots(context, self._device_ints(new_lens), self.block_table, self.free,
                            block_size=self.config.block_size, max_tokens=sum(new_lens))
        return Step(new_lens, slots, context, tuple(self.lens))

    def advance(self, step: Step, kept=None) -> None:
        """The step's tokens are the requests' now, or those that ``kept[r]`` names: pages of the rest go back.

        A number keeps the first so many, which is right for a chain. Of a tree a
        list names the accepted branch, from the root on, by its tokens' places in
        the step: its keys and values move to the places behind the request's
        last token, which its rotary positions (``depths``) have assumed already.
        """
        if step.lens is not None and list(step.lens) != self.lens:
            raise ValueError(f"the step was planned for requests of {list(step.lens)} tokens; they have {self.lens}")
        paths = []
        for k in step.new_lens if kept is None else kept:
            several = isinstance(k, (list, tuple, range)) or getattr(k, "ndim", 0)
            paths.append([int(i) for i in k] if several else list(range(int(k))) if int(k) >= 0 else [-1])
        if len(paths) != len(self.lens) or any(
                p and not (0 <= p[0] and p[-1] < n and all(a < b for a, b in zip(p, p[1:])))
                for p, n in zip(paths, step.new_lens)):
            raise ValueError(f"kept must be counts of at most {step.new_lens}, or rising places below them, got {kept}")
        moves = [(r, self.lens[r] + a, self.lens[r] + b) for r, p in enumerate(paths) for b, a in enumerate(p) if a != b]
        if moves:
            size = self.config.block_size
            rows, source, to = torch.tensor(moves, device=self.free.device).unbind(1)
            source_page, to_page = (self.block_table[rows, at // size].long() for at in (source, to))
            for pages in (self.k, self.v):
                pages[to_page, :, to % size] = pages[source_page, :, source % size]
        kept = [len(p) for p in paths]
        before, after, keep = self._pages([0] * len(kept)), self._pages(step.new_lens), self._pages(kept)
        free = self.free[sum(after) - sum(before):]
        back = [(r, c) for r in range(len(kept)) for c in range(keep[r], after[r])]
        if back:
            rows, columns = torch.tensor(back, device=free.device).unbind(1)
            free = torch.cat([self.block_table[rows, columns], free])
        self.free = free
        self.lens = [n + k for n, k in zip(self.lens, kept)]

    def release(self, request: int) -> None:
        """A finished request's pages go back, and its row is free for another. Between steps, not during one."""
        if not 0 <= request < len(self.lens):
            raise ValueError(f"request must be one of {len(self.lens)}, got {request}")
        pages = -(-self.lens[request] // self.config.block_size)
        self.free = torch.cat([self.free, self.block_table[request, :pages]])
        self.block_table[request] = -1
        self.lens[request] = 0


class ServingBlock(nn.Module):
    """Pre-norm decoder block with rotary positions, grouped heads and a bias + GELU MLP."""

    def __init__(self, config: ServingConfig | None = None, *, dtype: torch.dtype = torch.float16,
                 device: torch.device | str = "cuda") -> None:
        super().__init__()
        self.config = c = config if config is not None else ServingConfig()
        like = {"device": device, "dtype": dtype}
        self.attn_norm_weight = nn.Parameter(torch.ones(c.hidden, **like))
        self.mlp_norm_weight = nn.Parameter(torch.ones(c.hidden, **like))
        self.qkv_proj = nn.Linear(c.hidden, (c.heads + 2 * c.kv_heads) * c.head_dim, bias=False, **like)
        self.out_proj = nn.Linear(c.hidden, c.hidden, bias=False, **like)
        self.mlp_up = nn.Linear(c.hidden, c.intermediate, bias=True, **like)
        self.mlp_down = nn.Linear(c.intermediate, c.hidden, bias=False, **like)
        self.register_buffer("angles", rotary_table(c.max_positions, c.head_dim, base=c.rotary_base, device=device),
                             persistent=False)

    def _qkv(self, x: torch.Tensor):
        if x.ndim != 2 or x.shape[1] != self.config.hidden:
            raise ValueError(f"expected (tokens, {self.config.hidden}), got {tuple(x.shape)}")
        c = self.config
        normed = rmsnorm(x, self.attn_norm_weight, eps=c.eps)
        qkv = matmul(normed, self.qkv_proj.weight.t()).view(x.shape[0], c.heads + 2 * c.kv_heads, c.head_dim)
        return qkv[:, :c.heads], qkv[:, c.heads:c.heads + c.kv_heads], qkv[:, c.heads + c.kv_heads:]

    def _rest(self, x: torch.Tensor, mixed: torch.Tensor) -> torch.Tensor:
        x = x + matmul(mixed.reshape(x.shape), self.out_proj.weight.t())
        normed = rmsnorm(x, self.mlp_norm_weight, eps=self.config.eps)
        return x + matmul(fused_linear_gelu(normed, self.mlp_up.weight.t(), self.mlp_up.bias), self.mlp_down.weight.t())

    def prompts(self, x: torch.Tensor, cache: PagedCache, step: Step) -> torch.Tensor:
        """Whole prompts of requests that have no tokens yet, packed without padding."""
        if any(n and a for n, a in zip(cache.lens, step.new_lens)):
            raise ValueError("prompts() starts requests; tokens() continues them")
        q, k, v = self._qkv(x)
        turned = torch.empty(k.shape, dtype=k.dtype, device=k.device)
        q = rotary_to_cache(q, k, v, step.slots.positions, self.angles, cache.k, cache.v, step.slots.slots, k_out=turned)
        return self._rest(x, prefill_attention(q, turned, v, step.slots.cu_new))

    def tokens(self, x: torch.Tensor, cache: PagedCache, step: Step, tree_mask: torch.Tensor | None = None,
               depths: torch.Tensor | None = None) -> torch.Tensor:
        """New tokens of requests in the cache: chains, or trees given by ``tree_mask`` (:func:`tree_attention`)
        and, for their rotary positions, ``depths`` (int32: each token's distance below the request's last)."""
        q, k, v = self._qkv(x)
        positions = step.slots.positions
        if depths is not None:
            owner = torch.repeat_interleave(step.context_lens, step.slots.cu_new.diff(), output_size=x.shape[0])
            positions = owner + depths
        q = rotary_to_cache(q, k, v, positions, self.angles, cache.k, cache.v, step.slots.slots)
        one_each = all(n == 1 for n in step.new_lens) and tree_mask is None
        return self._rest(x, tree_attention(q, cache.k, cache.v, cache.block_table, step.context_lens,
                                            None if one_each else step.slots.cu_new, tree_mask))

"""Prompt attention and tree attention over a paged cache, against 64 bits.

Bounds are derived in attention_reference.py. Lengths of zero and one, odd
sizes, prompts that continue cached keys, rows that see nothing, grouped and
strided heads, what lies in masked and stale places, pages that end inside a
tile, masks of several words, long caches, other streams and graphs.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from kernelo_b200.kernels.attention import prefill_attention, tree_attention
from tests import attention_reference as ref

pytestmark = pytest.mark.gpu

HALF = (torch.float16, torch.bfloat16)
DTYPES = (*HALF, torch.float32)


def randn(gen, *shape, dtype, device, gain=1.0):
    return (torch.randn(*shape, generator=gen) * gain).to(dtype).to(device)


def offsets(lens, device):
    return torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device=device)


def prompt(lens_q, lens_k, heads, kv_heads, dim, dtype, device, seed=0, extra=0):
    gen = torch.Generator().manual_seed(seed)
    q = randn(gen, sum(lens_q) + extra, heads, dim, dtype=dtype, device=device, gain=2.0)
    k = randn(gen, sum(lens_k), kv_heads, dim, dtype=dtype, device=device)
    v = randn(gen, sum(lens_k), kv_heads, dim, dtype=dtype, device=device)
    return q, k, v, offsets(lens_q, device), offsets(lens_k, device)


def check_prompt(lens_q, lens_k, q, k, v, cu_q, cu_k, what, **kw):
    want, want_lse, bound, off = ref.packed(q, k, v, lens_q, lens_k, **kw)
    out, lse = prefill_attention(q, k, v, cu_q, cu_k, return_lse=True, **kw)
    assert out.dtype == q.dtype and lse.dtype == torch.float32
    ref.check(out, want, bound, what)
    ref.check_lse(lse, want_lse, off, what)
    return out, lse


# ------------------------------------------------------------------ prompts
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens", [(1,), (2,), (127,), (128,), (129,), (255, 1, 64), (257,), (0, 5, 0, 130, 0), (640,)])
def test_prompt_lengths(lens, dtype, device):
    check_prompt(lens, lens, *prompt(lens, lens, 4, 2, 64, dtype, device), f"{lens} {dtype}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [8, 16, 20, 32, 40, 64, 80, 112, 128, 136, 256])
def test_head_dimensions(dim, dtype, device):
    check_prompt((150, 77), (150, 77), *prompt((150, 77), (150, 77), 2, 1, dim, dtype, device), f"dim {dim} {dtype}")


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (7, 1), (8, 2), (32, 8)])
@pytest.mark.parametrize("causal", [True, False])
def test_grouped_heads(heads, kv_heads, causal, device):
    lens = (200, 333)
    check_prompt(lens, lens, *prompt(lens, lens, heads, kv_heads, 128, torch.bfloat16, device),
                 f"{heads}/{kv_heads} causal={causal}", causal=causal)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens_q,lens_k", [((5, 64, 1), (300, 64, 129)), ((128, 130), (1000, 131)),
                                           ((1,), (1,)), ((300,), (700,))])
def test_prompts_that_continue_cached_keys(lens_q, lens_k, dtype, device):
    check_prompt(lens_q, lens_k, *prompt(lens_q, lens_k, 4, 2, 128, dtype, device), f"{lens_q} {lens_k}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
def test_rows_without_keys_are_zero(dtype, causal, device):
    """More rows than keys (the first rows see none), no keys at all, rows of no request."""
    lens_q, lens_k = (200, 3, 140, 0), (50, 0, 130, 7)
    q, k, v, cu_q, cu_k = prompt(lens_q, lens_k, 4, 2, 64, dtype, device, extra=133)
    out, lse = check_prompt(lens_q, lens_k, q, k, v, cu_q, cu_k, f"{dtype}", causal=causal)
    empty = [*range(200, 203), *range(343, 476)] + (list(range(150)) + list(range(203, 213)) if causal else [])
    assert (out[empty] == 0).all() and (lse[empty] == -torch.inf).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_no_keys_anywhere(dtype, device):
    q = torch.randn(9, 2, 64, device=device).to(dtype)
    none = torch.empty(0, 1, 64, device=device, dtype=dtype)
    out, lse = prefill_attention(q, none, none, offsets([4, 5], device), offsets([0, 0], device), return_lse=True)
    assert (out == 0).all() and (lse == -torch.inf).all()
    out, lse = prefill_attention(q, none, none, offsets([], device), offsets([], device), return_lse=True)
    assert (out == 0).all() and (lse == -torch.inf).all()
    assert prefill_attention(q[:0], none, none, offsets([0], device)).shape == (0, 2, 64)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("poison", [float("nan"), float("inf"), float("-inf")])
def test_what_a_row_does_not_see_does_not_reach_it(dtype, poison, device):
    """Later tokens of the request, the next request's keys in the same tile, keys past the last request."""
    lens = (70, 90)
    q, k, v, cu_q, cu_k = prompt(lens, lens, 4, 2, 64, dtype, device)
    want, want_lse, bound, off = ref.packed(q, k, v, lens, lens)
    k, v = (torch.cat([t, torch.full_like(t[:40], poison)]) for t in (k, v))
    k[41:70], v[41:70] = poison, poison  # rows 0..40 see none of these, rows 41.. do
    out, lse = prefill_attention(q, k, v, cu_q, cu_k, return_lse=True)
    fine = [*range(41), *range(70, 160)]
    ref.check(out[fine], want[fine], bound[fine], f"{dtype} {poison}")
    ref.check_lse(lse[fine], want_lse[fine], off[fine], f"{dtype} {poison}")


@pytest.mark.parametrize("dtype", HALF)
def test_scores_far_apart_and_all_equal(dtype, device):
    """Scores that grow along the keys by hundreds (each tile raises the running maximum), then constant ones."""
    n, dim = 520, 64
    gen = torch.Generator().manual_seed(1)
    v = randn(gen, n, 1, dim, dtype=dtype, device=device)
    q = torch.zeros(n, 1, dim, device=device, dtype=dtype)
    k = torch.zeros(n, 1, dim, device=device, dtype=dtype)
    q[:, 0, 0] = 8.0
    k[:, 0, 0] = torch.arange(n, device=device) // 8  # exact in both types
    for case in (k, -k, torch.zeros_like(k)):
        check_prompt((n,), (n,), q, case, v, offsets([n], device), offsets([n], device), f"{dtype}", scale=1.0)


def test_scale_and_given_output(device):
    lens = (100, 31)
    q, k, v, cu_q, cu_k = prompt(lens, lens, 4, 4, 64, torch.float16, device)
    for scale in (0.0, 0.3, -0.1):
        check_prompt(lens, lens, q, k, v, cu_q, cu_k, f"scale {scale}", scale=scale)
    room = torch.full((131, 8, 80), 7.0, device=device, dtype=torch.float16)
    out = prefill_attention(q, k, v, cu_q, out=room[:, 2:6, 8:72])
    assert torch.equal(out, prefill_attention(q, k, v, cu_q))
    room[:, 2:6, 8:72] = 7.0
    assert (room == 7.0).all(), "written outside the output"


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("dim", [64, 128])
def test_views_of_one_projection(dim, dtype, device):
    """q, k and v as slices of one qkv row, and heads outermost."""
    lens = (300, 211)
    gen = torch.Generator().manual_seed(2)
    qkv = randn(gen, 511, 8, dim, dtype=dtype, device=device)
    cu = offsets(lens, device)
    q, k, v = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:]
    check_prompt(lens, lens, q, k, v, cu, cu, "qkv views")
    check_prompt(lens, lens, *(t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)), cu, cu, "heads first")
    odd = randn(gen, 511, 8, dim + 3, dtype=dtype, device=device)  # rows off the 16-byte grid
    check_prompt(lens, lens, *(odd[:, a:b, 1:1 + dim] for a, b in ((0, 4), (4, 6), (6, 8))), cu, cu, "odd rows")


def test_long_prompt_rows_sampled(device):
    """4100 tokens at 32/8 heads of 128: sampled rows of sampled heads."""
    n = 4100
    q, k, v, cu_q, cu_k = prompt((n,), (n,), 32, 8, 128, torch.bfloat16, device)
    out, lse = prefill_attention(q, k, v, cu_q, cu_k, return_lse=True)
    for h in (0, 13, 31):
        for rows in (slice(0, 130), slice(2040, 2060), slice(n - 130, n)):
            at = torch.arange(n, device=device)
            want, want_lse, bound, off = ref.attend(q[rows, h], k[:, h // 4], v[:, h // 4],
                                                    at[None, :] <= at[rows, None], 128 ** -0.5)
            ref.check(out[rows, h], want, bound, f"head {h}")
            ref.check_lse(lse[rows, h], want_lse, off, f"head {h}")


def test_the_same_inputs_give_the_same_bits(device):
    lens = (700, 900, 13)
    args = prompt(lens, lens, 8, 2, 128, torch.bfloat16, device)
    first = prefill_attention(*args)
    assert all(torch.equal(first, prefill_attention(*args)) for _ in range(5))


def test_prompt_on_another_stream_and_in_a_graph(device):
    lens = (100, 60)
    q, k, v, cu_q, cu_k = prompt(lens, lens, 4, 2, 64, torch.float16, device)
    want = prefill_attention(q, k, v, cu_q, cu_k)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = prefill_attention(q, k, v, cu_q, cu_k)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = prefill_attention(q, k, v, cu_q, cu_k)
    cu_q.copy_(offsets((60, 100), device))
    cu_k.copy_(cu_q)
    graph.replay()
    assert torch.equal(out, prefill_attention(q, k, v, cu_q, cu_k)) and not torch.equal(out, want)


def test_prompt_refusals(device):
    q, k, v, cu, _ = prompt((5,), (5,), 4, 2, 64, torch.float16, device)
    bad = [
        (dict(q=q[0]), "rows, heads, dim"), (dict(k=k[:, :, :32], v=v[:, :, :32]), "head dimension mismatch"),
        (dict(v=v[:4]), "k and v"), (dict(k=k.float(), v=v.float()), "dtype mismatch"),
        (dict(q=q[:, :3]), "not a multiple"), (dict(cu_q=cu.long()), "cu_q must be torch.int32"),
        (dict(cu_q=cu.cpu()), "cu_q must be on"), (dict(cu_q=cu[:0]), "requests"),
        (dict(cu_k=cu[:1]), "one shape"), (dict(q=q[:4]), "pass cu_k"),
        (dict(q=q.transpose(1, 2).contiguous().transpose(1, 2)), "contiguous last dimension"),
        (dict(out=q[:4]), "out must have shape"), (dict(out=q.float()), "dtype mismatch"),
        (dict(k=k.cpu(), v=v.cpu()), "one device"), (dict(scale=float("nan")), "finite"),
    ]
    for change, message in bad:
        args = dict(q=q, k=k, v=v, cu_q=cu) | change
        with pytest.raises(ValueError, match=message):
            prefill_attention(**args)
    wide = torch.zeros(5, 1, 264, device=device, dtype=torch.float16)
    with pytest.raises(ValueError, match="at most 256"):
        prefill_attention(wide, wide, wide, cu)


# ------------------------------------------------------------------ paged caches
def cache(context, nodes, heads, kv_heads, dim, block, dtype, device, *, seed=0, spare=3, columns=None, stale=None):
    """Queries, shuffled pages and the block table; slots past a request's end hold ``stale``."""
    gen, rng = torch.Generator().manual_seed(seed), np.random.default_rng(seed)
    blocks = [-(-(c + n) // block) for c, n in zip(context, nodes)]
    total = sum(blocks) + spare
    order = rng.permutation(total)
    table = np.full((len(context), columns or max([*blocks, 1])), -1, dtype=np.int32)
    k = randn(gen, total, kv_heads, block, dim, dtype=dtype, device=device)
    v = randn(gen, total, kv_heads, block, dim, dtype=dtype, device=device)
    at = 0
    for r, n in enumerate(blocks):
        table[r, :n] = order[at:at + n]
        at += n
        end = (context[r] + nodes[r]) % block
        if stale is not None and end:
            k[table[r, n - 1], :, end:], v[table[r, n - 1], :, end:] = stale, stale
    if stale is not None:
        k[torch.from_numpy(order[at:]).to(device)] = stale
        v[torch.from_numpy(order[at:]).to(device)] = stale
    q = randn(gen, sum(nodes), heads, dim, dtype=dtype, device=device, gain=2.0)
    return (q, k, v, torch.from_numpy(table).to(device),
            torch.tensor(context, dtype=torch.int32, device=device))


def random_trees(nodes, seed=0, words=1):
    """Per request the (n, n) mask of a random tree, and all rows' mask words."""
    rng = np.random.default_rng(seed)
    masks, rows = [], []
    for n in nodes:
        seen = np.zeros((n, n), dtype=bool)
        for i in range(n):
            if i and rng.random() < 0.9:
                seen[i] = seen[rng.integers(max(0, i - 5), i)]
            seen[i, i] = True
        masks.append(torch.from_numpy(seen))
        for i in range(n):
            value = sum(1 << int(j) for j in np.flatnonzero(seen[i]))
            rows.append([(value >> (64 * w)) & (2 ** 64 - 1) for w in range(words)])
    return masks, torch.from_numpy(np.array(rows, dtype=np.uint64).reshape(-1, words).view(np.int64))


def check_tree(context, nodes, q, k, v, table, lens, what, *, masks=None, words=None, cu=True, scale=None):
    want, want_lse, bound, off = ref.paged(q, k, v, table, context, nodes, masks, scale=scale)
    cu_q = offsets(nodes, q.device) if cu else None
    out, lse = tree_attention(q, k, v, table, lens, cu_q, None if words is None else words.to(q.device),
                              return_lse=True, scale=scale)
    ref.check(out, want, bound, what)
    ref.check_lse(lse, want_lse, off, what)
    return out, lse


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [16, 20, 32, 64, 80, 112, 128, 200, 256])
def test_one_token_each(dim, dtype, device):
    context = (0, 1, 15, 16, 63, 64, 65, 127, 128, 300)
    nodes = (1,) * len(context)
    check_tree(context, nodes, *cache(context, nodes, 4, 2, dim, 16, dtype, device), f"{dim} {dtype}", cu=False)


@pytest.mark.parametrize("block", [1, 3, 8, 16, 24, 64, 256])
@pytest.mark.parametrize("dtype", HALF)
def test_page_sizes(block, dtype, device):
    context, nodes = (0, 70, 200, 129), (1, 3, 5, 64)
    check_tree(context, nodes, *cache(context, nodes, 8, 2, 128, block, dtype, device, columns=300), f"block {block}")


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (5, 1), (8, 8), (16, 1), (32, 8), (40, 8), (24, 1)])
@pytest.mark.parametrize("count", [1, 4, 16, 33])
def test_trees_and_grouped_heads(heads, kv_heads, count, device):
    context, nodes = (100, 0, 257), (count, max(1, count // 2), count)
    masks, words = random_trees(nodes)
    check_tree(context, nodes, *cache(context, nodes, heads, kv_heads, 64, 16, torch.bfloat16, device),
               f"{heads}/{kv_heads} {count}", masks=masks, words=words)


@pytest.mark.parametrize("dtype", DTYPES)
def test_masks_of_several_words(dtype, device):
    context, nodes = (37, 300), (130, 65)
    masks, words = random_trees(nodes, words=3)
    check_tree(context, nodes, *cache(context, nodes, 4, 2, 64, 16, dtype, device), f"{dtype}", masks=masks, words=words)


@pytest.mark.parametrize("dtype", DTYPES)
def test_empty_requests_and_rows_that_see_nothing(dtype, device):
    """No context and an empty mask; requests without rows; rows of no request."""
    context, nodes = (0, 40, 0, 9), (3, 0, 2, 2)
    masks, words = random_trees(nodes)
    masks[0][1] = False
    words[1] = 0
    q, k, v, table, lens = cache(context, nodes, 4, 2, 64, 16, dtype, device)
    out, lse = check_tree(context, nodes, q, k, v, table, lens, f"{dtype}", masks=masks, words=words)
    assert (out[1] == 0).all() and (lse[1] == -torch.inf).all()
    extra = torch.cat([q, q[:2]])
    got, got_lse = tree_attention(extra, k, v, table, lens, offsets(nodes, device),
                                  torch.cat([words, words[:2]]).to(device), return_lse=True)
    assert torch.equal(got[:7], out) and (got[7:] == 0).all() and (got_lse[7:] == -torch.inf).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("stale", [float("nan"), float("inf")])
def test_stale_slots_and_masked_nodes_do_not_reach_a_row(dtype, stale, device):
    context, nodes = (3, 70, 130, 31), (5, 9, 1, 2)
    masks, words = random_trees(nodes, seed=3)
    args = cache(context, nodes, 8, 2, 64, 16, dtype, device, stale=stale)
    check_tree(context, nodes, *args, f"{dtype} {stale}", masks=masks, words=words)
    # the last node of request 1, seen by itself alone, holds what nobody else may meet
    q, k, v, table, lens = args
    masks[1][:8, 8] = False
    want, want_lse, bound, off = ref.paged(q, k, v, table, context, nodes, masks)
    place = 70 + 8
    page, at = int(table[1, place // 16]), place % 16
    k[page, :, at], v[page, :, at] = stale, stale
    out, lse = tree_attention(q, k, v, table, lens, offsets(nodes, device), words.to(device), return_lse=True)
    fine = [i for i in range(17) if i != 13]
    ref.check(out[fine], want[fine], bound[fine], "masked node")
    ref.check_lse(lse[fine], want_lse[fine], off[fine], "masked node")


@pytest.mark.parametrize("dtype", DTYPES)
def test_pages_the_table_does_not_name(dtype, device):
    """-1 and pages past the cache hold nothing; lengths past the table's row end with it."""
    context, nodes = (200, 60), (1, 1)
    q, k, v, table, lens = cache(context, nodes, 4, 2, 64, 16, dtype, device)
    table[0, 3], table[0, 7] = -1, k.shape[0]
    check_tree(context, nodes, q, k, v, table, lens, f"{dtype}", cu=False)
    check_tree(context, nodes, q, k, v, table[:, :2].contiguous(), lens, f"{dtype} short rows", cu=False)
    wide = torch.full((2, 40), -1, device=device, dtype=torch.int32)
    wide[:, 5:5 + table.shape[1]] = table
    check_tree(context, nodes, q, k, v, wide[:, 5:], lens, f"{dtype} strided table", cu=False)


@pytest.mark.parametrize("dtype", HALF)
def test_cache_layouts(dtype, device):
    """Slots outside heads, K and V in one tensor, and heads off the 16-byte grid."""
    context, nodes = (150, 33), (4, 7)
    q, k, v, table, lens = cache(context, nodes, 8, 2, 64, 16, dtype, device)
    base = check_tree(context, nodes, q, k, v, table, lens, "pages")[0]
    slots_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v)]
    assert torch.equal(check_tree(context, nodes, q, *slots_first, table, lens, "slots first")[0], base)
    both = torch.stack([k, v], 1)
    assert torch.equal(check_tree(context, nodes, q, both[:, 0], both[:, 1], table, lens, "one tensor")[0], base)
    odd = torch.zeros(*k.shape[:3], 67, device=device, dtype=dtype)
    odd[..., 1:65] = k
    check_tree(context, nodes, q, odd[..., 1:65], v, table, lens, "odd heads")


@pytest.mark.parametrize("nodes", [1, 7])
@pytest.mark.parametrize("dtype", HALF)
def test_long_cache_split_over_the_gpu(nodes, dtype, device):
    context, nodes = (33000, 5, 9001), (nodes,) * 3
    masks, words = random_trees(nodes)
    check_tree(context, nodes, *cache(context, nodes, 8, 2, 128, 32, dtype, device), f"{nodes}", masks=masks, words=words)


def test_more_requests_than_sms(device):
    rng = np.random.default_rng(0)
    context = tuple(int(c) for c in rng.integers(0, 90, 400))
    nodes = tuple(int(c) for c in rng.integers(0, 3, 400))
    check_tree(context, nodes, *cache(context, nodes, 4, 1, 32, 16, torch.float16, device), "400 requests")


def test_cache_offsets_past_32_bits(device):
    """Pages at the end of a cache of more than 2^32 elements."""
    block, dim = 16, 128
    pages = (2 ** 32) // (block * dim) + 40
    big = torch.empty(pages, 1, block, dim, device=device, dtype=torch.float16)
    context, nodes = (70, 200), (2, 1)
    q, k, v, table, lens = cache(context, nodes, 4, 1, dim, block, torch.float16, device)
    far = table + (pages - k.shape[0])
    big[pages - k.shape[0]:] = k
    want = tree_attention(q, k, k, table, lens, offsets(nodes, device))
    got = tree_attention(q, big, big, torch.where(table >= 0, far, -1).int(), lens, offsets(nodes, device))
    assert torch.equal(got, want)


def test_the_same_cache_gives_the_same_bits(device):
    context, nodes = (5000, 70, 3000), (1, 4, 9)
    q, k, v, table, lens = cache(context, nodes, 8, 2, 128, 16, torch.bfloat16, device)
    cu = offsets(nodes, device)
    first = tree_attention(q, k, v, table, lens, cu)
    assert all(torch.equal(first, tree_attention(q, k, v, table, lens, cu)) for _ in range(8))


def test_tree_on_two_streams_and_in_a_graph(device):
    context, nodes = (3000, 50), (1, 1)
    q, k, v, table, lens = cache(context, nodes, 8, 2, 128, 16, torch.float16, device)
    want = tree_attention(q, k, v, table, lens)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(tree_attention(q, k, v, table, lens))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = tree_attention(q, k, v, table, lens)
    lens.copy_(torch.tensor([17, 49], dtype=torch.int32))
    for _ in range(3):
        graph.replay()
    assert torch.equal(out, tree_attention(q, k, v, table, lens)) and not torch.equal(out, want)


def test_tree_refusals(device):
    context, nodes = (20, 5), (1, 1)
    q, k, v, table, lens = cache(context, nodes, 4, 2, 64, 16, torch.float16, device)
    cu, words = offsets(nodes, device), torch.ones(2, 1, dtype=torch.int64, device=device)
    bad = [
        (dict(q=q[0]), "rows, heads, dim"), (dict(k_cache=k[0], v_cache=v[0]), "pages"),
        (dict(v_cache=v[1:]), "pages"), (dict(q=q[:, :3]), "not a multiple"), (dict(q=q[..., :32]), "head dimension"),
        (dict(k_cache=k.bfloat16(), v_cache=v.bfloat16()), "dtype mismatch"),
        (dict(block_table=table.long()), "block_table must be int32"), (dict(block_table=table[0]), "block_table"),
        (dict(block_table=table.cpu()), "block_table must be on"), (dict(block_table=table.t().contiguous().t()), "rows"),
        (dict(context_lens=lens[:1]), "context_lens must have shape"), (dict(context_lens=lens.long()), "int32"),
        (dict(cu_q=cu[:2]), "cu_q must have shape"), (dict(cu_q=cu.long()), "cu_q must be"),
        (dict(q=torch.cat([q, q])), "pass cu_q"), (dict(tree_mask=words[:1]), "tree_mask must have shape"),
        (dict(tree_mask=words.int()), "tree_mask must be"), (dict(tree_mask=words[:, 0]), "tree_mask must have shape"),
        (dict(k_cache=k[:, :, :0], v_cache=v[:, :, :0]), "at least one token"), (dict(scale=float("inf")), "finite"),
    ]
    for change, message in bad:
        args = dict(q=q, k_cache=k, v_cache=v, block_table=table, context_lens=lens) | change
        with pytest.raises(ValueError, match=message):
            tree_attention(**args)


# ---------------------------------------------------- tiles in fp32 arithmetic
@pytest.mark.parametrize("block", [1, 3, 8, 24, 256])
@pytest.mark.parametrize("count", [1, 4, 20, 70])
@pytest.mark.parametrize("heads,kv_heads", [(5, 1), (8, 8), (32, 8)])
def test_fp32_trees(heads, kv_heads, count, block, device):
    """Both tile sizes; keys of a tile shared by up to 16 CTAs, and none; mask bits across blocks of 32 keys."""
    context, nodes = (33, 0, 700, 31), (count, 1, max(1, count - 1), max(1, count // 2))
    masks, words = random_trees(nodes, words=2)
    check_tree(context, nodes, *cache(context, nodes, heads, kv_heads, 64, block, torch.float32, device, columns=3000 // block),
               f"{heads}/{kv_heads} {count} {block}", masks=masks, words=words)


@pytest.mark.parametrize("dim", [24, 96, 128, 250])
def test_fp32_long_cache(dim, device):
    context, nodes = (5000,), (2,)
    args = cache(context, nodes, 4, 1, dim, 16, torch.float32, device, stale=float("nan"))
    out, lse = check_tree(context, nodes, *args, f"dim {dim}")
    q, k, v, table, lens = args
    again, again_lse = tree_attention(q, k, v, table, lens, offsets(nodes, device), return_lse=True)
    assert torch.equal(out, again) and torch.equal(lse, again_lse)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,kv_heads,dim", [(7, 1, 128), (3, 3, 33), (4, 2, 256)])
def test_fp32_prompts(heads, kv_heads, dim, causal, device):
    lens_q, lens_k = (333, 1, 64, 0, 90), (400, 1, 64, 5, 700)
    check_prompt(lens_q, lens_k, *prompt(lens_q, lens_k, heads, kv_heads, dim, torch.float32, device),
                 f"{heads}/{kv_heads} {dim} causal={causal}", causal=causal)


@pytest.mark.parametrize("dtype", DTYPES)
def test_elements_off_the_grid(dtype, device):
    """Rows that begin on odd elements, of odd lengths, and pages whose rows lie backwards in memory's order of heads."""
    lens = (70, 41)
    q, k, v, cu_q, cu_k = prompt(lens, lens, 4, 2, 77, dtype, device)
    q, k, v = (torch.nn.functional.pad(t, (1, 2))[:, :, 1:78] for t in (q, k, v))
    assert q.stride(1) == 80 and q.storage_offset() == 1
    check_prompt(lens, lens, q, k, v, cu_q, cu_k, f"{dtype}")
    context, nodes = (50, 7), (2, 1)
    q, k, v, table, at = cache(context, nodes, 4, 2, 77, 16, dtype, device)
    k, v = (torch.nn.functional.pad(t.transpose(1, 2).contiguous(), (1, 2))[..., 1:78].transpose(1, 2) for t in (k, v))
    check_tree(context, nodes, q, k, v, table, at, f"{dtype}")


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("requests", [3, 30, 31, 32, 40, 150])
def test_many_prompts_of_all_lengths(requests, causal, device):
    """More items than SMs, dealt out by their lengths or, for many requests, as they come; every row has to be there."""
    rng = np.random.default_rng(requests)
    lens_q = [int(n) for n in rng.choice([0, 1, 130, 256, 257, 600], requests)]
    lens_q[0] = 900
    lens_k = [n + int(m) for n, m in zip(lens_q, rng.choice([0, 0, 200], requests))]
    kv_heads = max(1, 150 // requests)
    check_prompt(lens_q, lens_k, *prompt(lens_q, lens_k, 2 * kv_heads, kv_heads, 32, torch.float16, device),
                 f"{requests} {causal}", causal=causal)

"""Attention where operands hold NaN, infinities or very large numbers.

What a row does not see must not reach it, and what it sees must: a NaN among a
row's scores or a score of +infinity makes the row NaN (infinity less infinity),
one of -infinity weighs nothing, whatever the key's place in its block and
however the work was cut. Finite rows are held to the bounds of
attention_reference.py.
"""

from __future__ import annotations

import pytest
import torch

from kernelo_b200.kernels.attention import prefill_attention, tree_attention
from kernelo_b200.runtime import native
from tests import attention_reference as ref
from tests.test_attention_gpu import DTYPES, HALF, cache, check_prompt, check_tree, offsets, prompt, random_trees

pytestmark = pytest.mark.gpu

LARGE = {torch.float16: 6e4, torch.bfloat16: 3e38, torch.float32: 3e38}


def check_rows(rows, got, lse, want, want_lse, bound, off, what):
    ref.check(got[rows], want[rows], bound[rows], what)
    ref.check_lse(lse[rows], want_lse[rows], off[rows], what)


# ------------------------------------------------------------------ prompts
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128])
def test_an_unseen_large_value_weighs_nothing(dim, dtype, device):
    """A later token's value of the type's largest size, at each place among eight keys, in the first and a later block."""
    lens = (300,)
    q, k, v, cu, _ = prompt(lens, lens, 2, 1, dim, dtype, device)
    want, want_lse, bound, off = ref.packed(q, k, v, lens, lens)
    for key in (*range(40, 48), *range(200, 208)):
        large = v.clone()
        large[key] = LARGE[dtype]
        out, lse = prefill_attention(q, k, large, cu, return_lse=True)
        check_rows(slice(0, key), out, lse, want, want_lse, bound, off, f"{dtype} key {key}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_a_seen_nan_key_makes_a_row_nan(causal, dim, dtype, device):
    lens = (300, 40)
    q, k, v, cu, _ = prompt(lens, lens, 2, 1, dim, dtype, device)
    want, want_lse, bound, off = ref.packed(q, k, v, lens, lens, causal=causal)
    for key in (*range(0, 8), *range(40, 48), *range(200, 208), 299):
        broken = k.clone()
        broken[key, 0, 3] = torch.nan
        out, lse = prefill_attention(q, broken, v, cu, causal=causal, return_lse=True)
        first = key if causal else 0
        assert out[first:300].isnan().all() and lse[first:300].isnan().all(), f"{dtype} key {key}"
        fine = [*range(first), *range(300, 340)]
        check_rows(fine, out, lse, want, want_lse, bound, off, f"{dtype} key {key}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128])
def test_infinite_scores_of_a_prompt(dim, dtype, device):
    """A key of +infinity in one element: NaN where the query's element is positive, no weight where it is negative."""
    lens = (300,)
    q, k, v, cu, _ = prompt(lens, lens, 2, 1, dim, dtype, device)
    q[:, :, 3] = torch.where(q[:, :, 3] == 0, torch.ones_like(q[:, :, 3]), q[:, :, 3])
    for key in (*range(0, 8), *range(200, 208)):
        broken = k.clone()
        broken[key, 0, 3] = torch.inf
        out, lse = prefill_attention(q, broken, v, cu, return_lse=True)
        at = torch.arange(300, device=device)
        for h in range(2):
            up = (at >= key) & (q[:, h, 3] > 0)
            assert out[up, h].isnan().all() and not (lse[up, h] < torch.inf).any(), f"{dtype} key {key}"
            seen = at[None, :] <= at[:, None]
            seen[:, key] = False  # a score of -infinity
            want, want_lse, bound, off = ref.attend(q[:, h], k[:, 0], v[:, 0], seen, dim ** -0.5)
            check_rows(~up, out[:, h], lse[:, h], want, want_lse, bound, off, f"{dtype} key {key}")


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_nan_query_of_a_prompt(dtype, device):
    lens = (300, 7)
    q, k, v, cu, _ = prompt(lens, lens, 4, 2, 64, dtype, device)
    want, want_lse, bound, off = ref.packed(q, k, v, lens, lens)
    rows = torch.tensor([0, 5, 130, 299, 303], device=device)
    q[rows, 1, 2] = torch.nan
    out, lse = prefill_attention(q, k, v, cu, return_lse=True)
    hit = torch.zeros(307, 4, dtype=torch.bool, device=device)
    hit[rows, 1] = True
    assert out[hit].isnan().all() and lse[hit].isnan().all()
    check_rows(~hit, out, lse, want, want_lse, bound, off, f"{dtype}")


# ------------------------------------------------------------------ paged caches
# (query heads, key heads, nodes): tiles of 16 rows and of 128; contexts that are cut over many CTAs and that are not
CUTS = [((33000,), 1), ((33000,), 16), ((20000, 40, 9001), 1), ((20000, 40, 9001), 9), ((50, 3), 2)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("context,count", CUTS)
def test_a_nan_query_over_a_cache(context, count, dtype, device):
    """The same answer whether the row's keys lie in one CTA's share or in many."""
    nodes = (count,) * len(context)
    masks, words = random_trees(nodes)
    q, k, v, table, lens = cache(context, nodes, 8, 2, 128, 32, dtype, device)
    want, want_lse, bound, off = ref.paged(q, k, v, table, context, nodes, masks)
    hit = torch.zeros(q.shape[:2], dtype=torch.bool, device=device)
    for r in range(len(context)):
        hit[r * count + count // 2, r % 8] = True
    q[..., 3] = torch.where(hit, torch.nan, q[..., 3].float()).to(dtype)
    out, lse = tree_attention(q, k, v, table, lens, offsets(nodes, device), words.to(device), return_lse=True)
    assert out[hit].isnan().all() and lse[hit].isnan().all()
    check_rows(~hit, out, lse, want, want_lse, bound, off, f"{dtype} {context} {count}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("count", [1, 16])
def test_a_stretch_of_nan_keys_in_a_long_cache(count, dtype, device):
    """Whole shares of the cache in which every score is NaN, and a single key; other requests are untouched."""
    context, nodes = (33000, 500), (count, count)
    masks, words = random_trees(nodes)
    q, k, v, table, lens = cache(context, nodes, 8, 2, 128, 32, dtype, device)
    want, want_lse, bound, off = ref.paged(q, k, v, table, context, nodes, masks)
    for pages in (slice(300, 700), slice(500, 501)):
        broken = k.clone()
        broken[table[0, pages].long(), 1] = torch.nan  # of the second key head
        out, lse = tree_attention(q, broken, v, table, lens, offsets(nodes, device), words.to(device), return_lse=True)
        assert out[:count, 4:].isnan().all() and lse[:count, 4:].isnan().all()
        hit = torch.zeros(q.shape[:2], dtype=torch.bool, device=device)
        hit[:count, 4:] = True
        check_rows(~hit, out, lse, want, want_lse, bound, off, f"{dtype} {pages}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("count", [1, 16])
def test_infinite_scores_over_a_cache(count, dtype, device):
    context, nodes = (9000, 60), (count, count)
    q, k, v, table, lens = cache(context, nodes, 8, 2, 128, 16, dtype, device)
    masks = [torch.ones(count, count, dtype=torch.bool).tril() for _ in nodes]
    q[..., 3] = torch.where(q[..., 3] == 0, torch.ones_like(q[..., 3]), q[..., 3])
    broken = k.clone()
    for r, place in ((0, 4001), (1, 38)):
        broken[table[r, place // 16].long(), :, place % 16, 3] = torch.inf
    out, lse = tree_attention(q, broken, v, table, lens, offsets(nodes, device), return_lse=True)
    up = q[..., 3] > 0
    assert out[up].isnan().all() and not (lse[up] < torch.inf).any()
    for r, place in ((0, 4001), (1, 38)):
        at = torch.arange(context[r] + count, device=device)
        page = table[r].long()[at // 16]
        seen = torch.ones(count, context[r] + count, dtype=torch.bool, device=device)
        seen[:, context[r]:] = masks[r].to(device)
        seen[:, place] = False
        rows = slice(r * count, (r + 1) * count)
        for h in range(8):
            want, want_lse, bound, off = ref.attend(q[rows, h], k[page, h // 4, at % 16], v[page, h // 4, at % 16], seen,
                                                    128 ** -0.5)
            check_rows(~up[rows, h], out[rows, h], lse[rows, h], want, want_lse, bound, off, f"{dtype} head {h}")


# ------------------------------------------------------- rows computed again
def check_columns(got, want, bound, column, what):
    """Every column but `column`, in which a seen value is infinite."""
    keep = [e for e in range(got.shape[-1]) if e != column]
    ref.check(got[..., keep], want[..., keep], bound[..., keep], what)
    assert not got[..., column].isfinite().any(), what


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("count", [1, 16])
def test_an_infinite_value_that_long_requests_see(count, dtype, device):
    """Only the column that the rows see it in is not finite; other requests lose nothing."""
    context, nodes = (131072, 300, 40), (count,) * 3
    masks, words = random_trees(nodes)
    q, k, v, table, lens = cache(context, nodes, 8, 2, 128, 32, dtype, device)
    want, want_lse, bound, off = ref.paged(q, k, v, table, context, nodes, masks)
    v[table[0, 5].long(), 0, 7, 9] = torch.inf  # of the first key head
    native.device_status()
    out, lse = tree_attention(q, k, v, table, lens, offsets(nodes, device), words.to(device), return_lse=True)
    assert native.device_status() == 0
    check_columns(out[:count, :4], want[:count, :4], bound[:count, :4], 9, f"{dtype}")
    ref.check_lse(lse, want_lse, off, f"{dtype}")
    ref.check(out[count:], want[count:], bound[count:], f"{dtype}")
    ref.check(out[:count, 4:], want[:count, 4:], bound[:count, 4:], f"{dtype}")


@pytest.mark.parametrize("dtype", HALF)
def test_an_infinite_value_that_a_long_prompt_sees(dtype, device):
    lens = (40000, 500)
    q, k, v, cu, _ = prompt(lens, lens, 1, 1, 64, dtype, device)
    v[3, 0, 9] = torch.inf
    native.device_status()
    out, lse = prefill_attention(q, k, v, cu, return_lse=True)
    assert native.device_status() == 0
    at = torch.arange(40000, device=device)
    clean = v.clone()
    clean[3, 0, 9] = 0.0
    for rows in (slice(3, 130), slice(20000, 20100), slice(39900, 40000)):
        want, want_lse, bound, off = ref.attend(q[rows, 0], k[:40000, 0], clean[:40000, 0], at[None, :] <= at[rows, None], 0.125)
        check_columns(out[rows, 0], want, bound, 9, f"{dtype} {rows}")
        ref.check_lse(lse[rows, 0], want_lse, off, f"{dtype} {rows}")
    want, want_lse, bound, off = ref.packed(q[40000:], k[40000:], v[40000:], (500,), (500,))
    ref.check(out[40000:], want, bound, f"{dtype}")
    ref.check_lse(lse[40000:], want_lse, off, f"{dtype}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("count", [2, 16])
def test_an_infinite_value_of_one_node_over_a_long_cache(count, dtype, device):
    """The other nodes' rows are computed again, which takes its time: the waits beside it do not run out, and
    neither these rows nor other requests lose anything."""
    context, nodes = (131072, 300, 40), (count,) * 3
    masks, words = random_trees(nodes)
    for r in range(3):
        masks[r][:, count - 1] = torch.arange(count) == count - 1
    q, k, v, table, lens = cache(context, nodes, 8, 2, 128, 32, dtype, device)
    want, want_lse, bound, off = ref.paged(q, k, v, table, context, nodes, masks)
    place = context[0] + count - 1
    v[table[0, place // 32].long(), :, place % 32, 9] = torch.inf
    native.device_status()
    out, lse = tree_attention(q, k, v, table, lens, offsets(nodes, device), words.to(device), return_lse=True)
    assert native.device_status() == 0
    fine = [i for i in range(3 * count) if i != count - 1]
    check_rows(fine, out, lse, want, want_lse, bound, off, f"{dtype}")
    check_columns(out[count - 1], want[count - 1], bound[count - 1], 9, f"{dtype}")


@pytest.mark.parametrize("dtype", HALF)
def test_an_infinite_value_at_the_end_of_a_long_prompt(dtype, device):
    lens = (40000, 500)
    q, k, v, cu, _ = prompt(lens, lens, 1, 1, 64, dtype, device)
    clean = v.clone()
    v[39999, 0, 9] = torch.inf
    native.device_status()
    out, lse = prefill_attention(q, k, v, cu, return_lse=True)
    assert native.device_status() == 0
    at = torch.arange(40000, device=device)
    for rows in (slice(0, 130), slice(39700, 39800), slice(39900, 39999)):
        want, want_lse, bound, off = ref.attend(q[rows, 0], k[:40000, 0], clean[:40000, 0], at[None, :] <= at[rows, None], 0.125)
        ref.check(out[rows, 0], want, bound, f"{dtype} {rows}")
        ref.check_lse(lse[rows, 0], want_lse, off, f"{dtype} {rows}")
    assert not out[39999, 0, 9].isfinite() and out[39999, 0, :9].isfinite().all()
    want, want_lse, bound, off = ref.packed(q[40000:], k[40000:], v[40000:], (500,), (500,))
    ref.check(out[40000:], want, bound, f"{dtype}")


# --------------------------------------------------------- large values, seen
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128])
def test_a_seen_large_value_of_a_prompt(dim, dtype, device):
    """One value of the type's largest size times weights of up to one stays finite, as the result does."""
    lens = (300,)
    q, k, v, cu, _ = prompt(lens, lens, 2, 1, dim, dtype, device)
    for key in (0, 5, *range(128, 136), 200, 290):
        large = v.clone()
        large[key] = LARGE[dtype]
        check_prompt(lens, lens, q, k, large, cu, cu, f"{dtype} key {key}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("context,count", CUTS)
def test_a_seen_large_value_of_a_cache(context, count, dtype, device):
    nodes = (count,) * len(context)
    masks, words = random_trees(nodes)
    q, k, v, table, lens = cache(context, nodes, 8, 2, 128, 32, dtype, device)
    for place in (0, 40, context[0] // 2, context[0]):
        large = v.clone()
        for r, c in enumerate(context):
            at = min(place, c)
            large[table[r, at // 32].long(), :, at % 32] = LARGE[dtype]
        check_tree(context, nodes, q, k, large, table, lens, f"{dtype} {context} {count} {place}", masks=masks, words=words)

"""Operands that stand for several: key heads, pages and query heads expanded from one (strides of zero)."""

from __future__ import annotations

import pytest

from tests.test_attention_gpu import DTYPES, cache, check_prompt, check_tree, prompt

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
def test_expanded_heads_of_a_prompt(dtype, device):
    lens = (150, 33)
    q, k, v, cu, _ = prompt(lens, lens, 4, 2, 64, dtype, device)
    check_prompt(lens, lens, q[:, :1].expand(-1, 4, -1), k[:, :1].expand(-1, 2, -1), v[:, 1:].expand(-1, 2, -1), cu, cu,
                 f"{dtype}")
    check_prompt(lens, lens, q, k[:1].expand(183, -1, -1), v, cu, cu, f"{dtype} one key")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("count", [1, 16])
def test_expanded_heads_and_pages_of_a_cache(count, dtype, device):
    context, nodes = (500, 70), (count, count)
    q, k, v, table, lens = cache(context, nodes, 8, 2, 64, 16, dtype, device)
    check_tree(context, nodes, q, k[:, :1].expand(-1, 2, -1, -1), v, table, lens, f"{dtype} heads")
    check_tree(context, nodes, q, k[:1].expand(k.shape), v[:1].expand(v.shape), table, lens, f"{dtype} pages")
    check_tree(context, nodes, q, k, v[:, :, :1].expand(v.shape), table, lens, f"{dtype} slots")
    check_tree(context, nodes, q[:, :1].expand(-1, 8, -1), k, v, table, lens, f"{dtype} queries")

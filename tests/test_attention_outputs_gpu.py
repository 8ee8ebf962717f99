"""Outputs given by the caller: beside the operands in one buffer, and refused on top of them or of themselves."""

from __future__ import annotations

import pytest
import torch

from kernelo_b200.kernels.attention import prefill_attention, tree_attention
from tests.test_attention_gpu import DTYPES, cache, offsets, prompt

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
def test_prompt_output(dtype, device):
    lens = (150, 33)
    q, k, v, cu, _ = prompt(lens, lens, 4, 2, 64, dtype, device)
    want = prefill_attention(q, k, v, cu)
    buf = torch.cat([q, k, v, torch.zeros_like(q)], 1)
    q, k, v, out = buf.split([4, 2, 2, 4], 1)
    assert torch.equal(prefill_attention(q, k, v, cu, out=out), want) and torch.equal(out, want)
    for given, message in ((q, "memory with q"), (buf[:, 2:6], "memory with q"), (buf[:, 4:8], "memory with k"),
                           (buf[:, 7:11], "memory with v"), (out[:1].expand_as(out), "itself"),
                           (out[:, :1].expand_as(out), "itself")):
        with pytest.raises(ValueError, match=message):
            prefill_attention(q, k, v, cu, out=given)


@pytest.mark.parametrize("dtype", DTYPES)
def test_tree_output(dtype, device):
    context, nodes = (500, 70), (3, 2)
    q, k, v, table, lens = cache(context, nodes, 4, 2, 64, 16, dtype, device)
    cu = offsets(nodes, device)
    want = tree_attention(q, k, v, table, lens, cu)
    out = torch.zeros_like(q)
    assert torch.equal(tree_attention(q, k, v, table, lens, cu, out=out), want)
    for given, message in ((q, "memory with q"), (k.view(-1, 4, 64)[:5], "memory with k_cache"),
                           (v.view(-1, 4, 64)[-5:], "memory with v_cache"), (out[:1].expand_as(out), "itself")):
        with pytest.raises(ValueError, match=message):
            tree_attention(q, k, v, table, lens, cu, out=given)

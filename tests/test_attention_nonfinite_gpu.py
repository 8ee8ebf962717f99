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

from kernelo_b200.kernels.attention import prefill_attention
from tests import attention_reference as ref
from tests.test_attention_gpu import DTYPES, prompt

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

"""Softmax of rows in which a mask has left little: most elements, whole vectors and whole threads are -inf.

The gate's bound: exponentials are off by at most 2^-22 and rescaled once, sums by a few 2^-24 of positive terms, and the
result is rounded to its type: below 2^-18 and half a unit, relative.
"""

from __future__ import annotations

import pytest
import torch

from kernelo_b200.kernels.softmax import softmax

pytestmark = pytest.mark.gpu

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


@pytest.mark.parametrize("dtype", list(UNIT))
@pytest.mark.parametrize("rows", [5, 700])
@pytest.mark.parametrize("cols", [7, 501, 512, 1000, 4097, 8192, 32000, 32001, 65536])
def test_rows_that_a_mask_leaves_little_of(cols, rows, dtype, device):
    gen = torch.Generator(device=device).manual_seed(0)
    x = (torch.randn(rows, cols, generator=gen, device=device) * 4).to(dtype)
    x[1] = -torch.inf
    x[1, cols // 2] = 3.0
    x[2, cols // 3:] = -torch.inf
    x[3, :-1] = -torch.inf
    x[4] = -torch.inf  # nothing left: zeros, as attention gives for a row that sees no key
    got = softmax(x)
    want = x.double().softmax(-1)
    want[4] = 0.0
    tiny = 2.0 ** -24 if dtype == torch.float16 else 2.0 ** -126  # smaller results may be flushed or lose bits
    assert ((got.double() - want).abs() <= (2.0 ** -18 + UNIT[dtype]) * want + tiny).all()
    assert got[1, cols // 2] == 1 and got[3, -1] == 1

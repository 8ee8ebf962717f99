"""Softmax of rows that have no probabilities: a NaN, or an infinity above all others, shows at every element, whichever
threads have nothing but -inf. (Each element is its exponential over a sum that is NaN.)"""

from __future__ import annotations

import pytest
import torch

from kernelo_b200.kernels.softmax import softmax

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [6, 700])
@pytest.mark.parametrize("cols", [7, 501, 512, 1000, 4097, 8192, 32000, 32001, 65536])
@pytest.mark.parametrize("bad", [torch.nan, torch.inf])
def test_a_bad_element_shows_in_its_whole_row(bad, cols, rows, dtype, device):
    gen = torch.Generator(device=device).manual_seed(0)
    x = torch.randn(rows, cols, generator=gen, device=device).to(dtype)
    x[1:5] = -torch.inf
    x[1, cols // 3] = bad  # nothing else
    x[2, 0], x[2, cols - 1] = bad, 1.0
    x[3, 0], x[3, cols // 2] = 1.0, bad  # in a thread that has nothing else
    x[4, :cols // 2], x[4, cols // 4] = 2.0, bad
    got = softmax(x)
    assert got[1:5].isnan().all()
    assert not got[0].isnan().any() and not got[5:].isnan().any()

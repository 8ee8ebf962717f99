"""What head norms refuse by the numbers and the memory that they are given, without a GPU."""

from __future__ import annotations

import math

import pytest
import torch

from kernelo_b200.kernels.rotary import _check_norm
from kernelo_b200.runtime import native
from tests.test_serving_step_host import packed, refused


@pytest.mark.parametrize("eps", [1e-46, 1e-40, 2.0 ** -127, 3.5e38, 1e300, 0.0, -1e-5, math.inf, math.nan])
def test_an_eps_that_fp32_does_not_hold_is_refused(eps):
    lib, heads = native.load(), dict(heads=4, kv_heads=2, dim=64)
    refused(lib.kf_norm_rotary, "kf_norm_rotary_args", native.KF_ERR_INVALID_ARGUMENT, "eps", **heads, eps=eps)
    refused(lib.kf_norm_rotary_grad, "kf_norm_rotary_grad_args", native.KF_ERR_INVALID_ARGUMENT, "eps", **heads, eps=eps)
    q, w = torch.zeros(1, 2, 64), torch.ones(64)
    with pytest.raises(ValueError, match="eps must be positive"):
        _check_norm(q, w, w, eps)


@pytest.mark.parametrize("eps", [2.0 ** -126, 1e-12, 1e-5, 1.0, 3.4e38])
def test_an_eps_that_fp32_holds_is_taken(eps):
    args = packed("kf_norm_rotary_args", heads=4, kv_heads=2, dim=64, eps=eps)  # of no tokens
    assert native.load().kf_norm_rotary(args, None) == native.KF_OK
    q, w = torch.zeros(1, 2, 64), torch.ones(64)
    _check_norm(q, w, w, eps)

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


# The addresses are made up, so calls that pass the checks must end for want of a device.
no_device = pytest.mark.skipif(torch.cuda.is_available(), reason="made-up addresses, for hosts without a device")

Q, K, V, OUT, CACHE = (0x10000000 * i for i in range(1, 6))
HEADS = dict(dtype=native.native_code(torch.bfloat16), tokens=10, heads=4, kv_heads=1, dim=64, eps=1e-5, rot=32, table_rows=100,
             q=Q, sq_row=448, sq_head=64, q_out=OUT, sqo_row=256, sqo_head=64, k=Q + 512, sk_row=448, sk_head=64,
             k_out=OUT + 0x100000, sko_row=64, sko_head=64, positions=0x8000, table=0x20000, q_weight=0x3000, k_weight=0x4000)
CACHED = dict(v=Q + 640, sv_row=448, sv_head=64, k_cache=CACHE, skc_page=2048, skc_head=1024, skc_slot=64, v_cache=CACHE + 2048,
              svc_page=2048, svc_head=1024, svc_slot=64, pages=7, block_size=16, slots=0x6000)  # a page's keys, then its values
LOGITS = dict(dtype=native.native_code(torch.float32), logits=Q, s_row=1000, out=OUT, so_row=1040, rows=6, vocab=1000, tokens=K, st_row=20,
              token_cols=20, token_lens=0x3000, repetition=0x3100, frequency=0x3200, presence=0x3300, prompt_lens=0x3400,
              bias_tokens=V, sb_row=8, bias_values=0x9000, sv_row=8, bias_cols=8, allowed=0xa000, sa_row=32, masks=3,
              allowed_rows=0x3500)


@no_device
@pytest.mark.parametrize("change,message", [
    (dict(q_out=Q + 128), "q_out shares memory with q"),
    (dict(q_out=Q, sqo_row=448, tokens=9, k=Q + 510), "q_out shares memory with k"),
    (dict(q_out=0x3000 - 10 * 512 + 2), "q_out shares memory with q_weight"),
    (dict(k_out=0x4000 + 126), "k_out shares memory with k_weight"),
    (dict(q_out=0x8000 + 36), "q_out shares memory with positions"),
    (dict(k_out=0x20000 + 12000), "k_out shares memory with table"),
    (dict(k_out=OUT + 5118), "k_out shares memory with q_out"),
    (dict(q_out=OUT, sqo_row=192), "q_out overlaps itself"),
    (dict(CACHED, k_out=0x6000 + 72), "k_out shares memory with slots"),
    (dict(CACHED, k_cache=Q + 1000), "k_cache shares memory with q"),
    (dict(CACHED, v_cache=CACHE + 2046), "v_cache shares memory with k_cache"),
    (dict(CACHED, v_cache=CACHE + 4096 + 2046), "v_cache shares memory with k_cache"),
    (dict(CACHED, v_cache=OUT + 4000), "v_cache shares memory with q_out"),
    (dict(CACHED, k_cache=0x3000), "k_cache shares memory with q_weight"),
    (dict(CACHED, skc_slot=0), "k_cache overlaps itself"),
    (dict(CACHED, svc_page=0), "v_cache overlaps itself"),
])
def test_outputs_that_share_memory_are_refused(change, message):
    refused(native.load().kf_norm_rotary, "kf_norm_rotary_args", native.KF_ERR_INVALID_ARGUMENT, message, **(HEADS | change))


@no_device
@pytest.mark.parametrize("change,message", [
    (dict(out=Q + 4), "out shares memory with logits"), (dict(out=Q), "out shares memory with logits"),
    (dict(so_row=999), "out overlaps itself"),
    (dict(out=K + 476), "out shares memory with tokens"), (dict(out=0x3000 + 20), "out shares memory with token_lens"),
    (dict(token_lens=OUT + 3998, prompt_lens=0), "out shares memory with token_lens"),
    (dict(prompt_lens=OUT + 500), "prompt_lens"), (dict(repetition=OUT + 500), "repetition"),
    (dict(frequency=OUT + 500), "frequency"), (dict(presence=OUT + 500), "presence"), (dict(bias_tokens=OUT + 500), "bias_tokens"),
    (dict(bias_values=OUT + 4000, sv_row=1040, bias_cols=41), "bias_values"), (dict(allowed=OUT + 500), "with allowed"),
    (dict(allowed_rows=OUT + 500), "allowed_rows"),
])
def test_logits_that_share_memory_are_refused(change, message):
    refused(native.load().kf_adjust_logits, "kf_logits_args", native.KF_ERR_INVALID_ARGUMENT, message, **(LOGITS | change))


@no_device
def test_outputs_of_their_own_pass_the_checks():
    in_place = dict(q_out=Q, sqo_row=448, k_out=Q + 512, sko_row=448)
    for change in ({}, in_place, CACHED, CACHED | in_place, CACHED | dict(k_out=0), CACHED | dict(v_cache=CACHE + 0x100000),
                   dict(q_out=0x3000 - 10 * 512), dict(k_out=0x4000 + 128), dict(tokens=1, q_out=Q + 640),
                   dict(kv_heads=0, k=0, k_out=0x3000), dict(rot=0, table=OUT, positions=OUT)):
        args = packed("kf_norm_rotary_args", **(HEADS | change))
        assert native.load().kf_norm_rotary(args, None) not in (native.KF_OK, native.KF_ERR_INVALID_ARGUMENT), change
    for change in (dict(out=Q, so_row=1000), {}, dict(bias_values=OUT + 4000, sv_row=1040, bias_cols=40), dict(rows=1, out=Q),
                   dict(tokens=0, token_lens=OUT), dict(allowed=0, allowed_rows=OUT), dict(bias_tokens=0, bias_values=OUT)):
        args = packed("kf_logits_args", **(LOGITS | change))
        assert native.load().kf_adjust_logits(args, None) not in (native.KF_OK, native.KF_ERR_INVALID_ARGUMENT), change

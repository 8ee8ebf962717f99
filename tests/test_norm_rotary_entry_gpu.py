"""The entries of head norms and logits: heads of one kind alone and no weight for the other, and outputs that lie among
other memory."""

from __future__ import annotations

import pytest
import torch

from kernelo_b200.kernels.logits import adjust_logits
from kernelo_b200.kernels.rotary import norm_rotary, norm_rotary_to_cache, rotary_table
from kernelo_b200.runtime import native
from tests.test_norm_rotary_gpu import inputs
from tests.test_serving_step_host import packed

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads", [1, 5, 18, 37])  # the last ones leave lanes of a warp without a head
@pytest.mark.parametrize("tokens", [1, 3, 700])
def test_heads_of_one_kind_without_the_other_weight(tokens, heads, dtype, device):
    x, none, _, w, _, positions = inputs(tokens, heads, 0, 128, dtype, device)
    table = rotary_table(5000, 128, device=device)
    want, _ = norm_rotary(x, none, positions, table, w, w)
    common = dict(dtype=native.native_code(dtype), positions=positions.data_ptr(), table=table.data_ptr(),
                  table_rows=5000, rot=128, tokens=tokens, dim=128, eps=1e-5)
    for kind in "qk":
        out = torch.full_like(x, torch.nan)
        fields = {kind: x.data_ptr(), f"s{kind}_row": x.stride(0), f"s{kind}_head": x.stride(1), f"{kind}_out": out.data_ptr(),
                  f"s{kind}o_row": out.stride(0), f"s{kind}o_head": out.stride(1), f"{kind}_weight": w.data_ptr(),
                  "heads" if kind == "q" else "kv_heads": heads}
        args = packed("kf_norm_rotary_args", **common, **fields)
        assert native.load().kf_norm_rotary(args, native.current_stream_handle(device)) == native.KF_OK, native.last_error()
        assert torch.equal(out, want)


def test_outputs_among_other_memory(device):
    """A projection of one key head turned in place, keys and values of each page side by side, and what is refused of them."""
    tokens, dim = 33, 64
    qkv = torch.randn(tokens, 6, dim, device=device).half()
    w = torch.randn(3, dim, device=device).half()
    table = rotary_table(100, dim, device=device)
    positions = torch.arange(tokens, dtype=torch.int32, device=device)
    slots = torch.randperm(48, device=device)[:tokens]
    pages = torch.zeros(3, 2, 1, 16, dim, device=device, dtype=torch.float16)
    q, k, v = qkv[:, :4], qkv[:, 4:5], qkv[:, 5:]
    want_q, want_k = norm_rotary(q, k, positions, table, w[0], w[1])
    value = v.clone()
    operands = (positions, table, w[0], w[1], pages[:, 0], pages[:, 1], slots)
    for bad, name in ((dict(k_out=v), "k_out shares memory with v"),
                      (dict(k_out=pages.view(-1, 1, dim)[:tokens]), "k_out shares memory with k_cache")):
        with pytest.raises(ValueError, match=name):
            norm_rotary_to_cache(q, k, v, *operands, **bad)
    flat = torch.zeros(tokens * dim + dim, device=device, dtype=torch.float16)
    with pytest.raises(ValueError, match="k_out shares memory with k_weight"):
        norm_rotary_to_cache(q, k, v, positions, table, w[0], flat[tokens * dim - dim:tokens * dim], *operands[4:],
                             k_out=flat[:tokens * dim].view(tokens, 1, dim))
    with pytest.raises(ValueError, match="v_cache shares memory with k_cache"):
        norm_rotary_to_cache(q, k, v, *operands[:4], pages[:, 0], pages[:, 0], slots)
    assert torch.equal(qkv[:, 5:], value) and not pages.any()
    assert norm_rotary_to_cache(q, k, v, *operands, q_out=q, k_out=k) is q
    assert torch.equal(q, want_q) and torch.equal(k, want_k)
    assert torch.equal(pages[slots // 16, 0, :, slots % 16], want_k) and torch.equal(pages[slots // 16, 1, :, slots % 16], value)


def test_logits_among_other_memory(device):
    """Biases behind the logits in one buffer, and an output that would take them."""
    buf = torch.randn(5, 640, device=device)
    tokens = torch.randint(0, 600, (5, 40), device=device, dtype=torch.int32)
    before = buf.clone()
    want = adjust_logits(buf[:, :600].clone(), bias_tokens=tokens, bias_values=buf[:, 600:].clone())
    with pytest.raises(ValueError, match="out shares memory with bias_values"):
        adjust_logits(torch.zeros(5, 601, device=device), bias_tokens=tokens, bias_values=buf[:, 600:], out=buf[:, :601])
    assert torch.equal(buf, before)
    got = adjust_logits(buf[:, :600], bias_tokens=tokens, bias_values=buf[:, 600:], out=buf[:, :600])
    assert torch.equal(got, want) and torch.equal(buf[:, 600:], before[:, 600:])

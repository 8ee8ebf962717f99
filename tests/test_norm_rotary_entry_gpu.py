"""The C entry of head norms with heads of one kind alone and no weight for the other, beside the Python call that has both."""

from __future__ import annotations

import pytest
import torch

from kernelo_b200.kernels.rotary import norm_rotary, rotary_table
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

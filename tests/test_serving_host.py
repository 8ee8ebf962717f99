"""The serving operators' host side, without a GPU: argument structs against the
header, refusals that need no device, rotary tables."""

from __future__ import annotations

import math
import re
from pathlib import Path

import pytest
import torch

from kernelo_b200.kernels import attention
from kernelo_b200.kernels.attention import prefill_attention, tree_attention
from kernelo_b200.kernels.paged import build_slots
from kernelo_b200.kernels.rotary import rotary, rotary_table
from kernelo_b200.runtime import native

HEADER = Path(__file__).resolve().parent.parent / "include" / "kernelo_b200.h"


@pytest.mark.parametrize("name,packed", [("kf_prefill_args", native.PREFILL_ARGS), ("kf_tree_args", native.TREE_ARGS),
                                         ("kf_rotary_args", native.ROTARY_ARGS), ("kf_slots_args", native.SLOTS_ARGS)])
def test_argument_structs_match_the_header(name, packed):
    """Every field is 8 bytes wide, in the header's order; the only doubles are the scales."""
    body = re.search(r"typedef struct %s \{(.*?)\}" % name, HEADER.read_text(), re.S).group(1)
    fields = []
    for line in filter(str.strip, body.split(";")):
        kind = "d" if line.strip().startswith("double") else "q"
        assert kind == "d" or "*" in line or line.strip().startswith("int64_t"), line
        fields += [kind] * len(line.split(","))
    letters = "".join(c * int(n or 1) for n, c in re.findall(r"(\d*)([a-z])", packed.format))
    assert letters == "".join(fields) and packed.size == 8 * len(fields)


def test_c_entries_refuse_before_touching_a_device():
    lib = native.load()
    for entry in (lib.kf_prefill_attention, lib.kf_tree_attention, lib.kf_rotary, lib.kf_build_slots):
        assert entry(None, None) == native.KF_ERR_INVALID_ARGUMENT
    zeros = dict(PREFILL_ARGS=lib.kf_prefill_attention, ROTARY_ARGS=lib.kf_rotary, SLOTS_ARGS=lib.kf_build_slots)
    for name, entry in zeros.items():
        packed = getattr(native, name)
        count = packed.size // 8
        assert entry(packed.pack(*[9] + [0] * (count - 1)), None) == native.KF_ERR_INVALID_ARGUMENT, name
        assert native.last_error()
    # rows without data are nothing to do; a head that does not divide, or is too wide, is refused
    def prefill(**fields):
        names = ("dtype q sq_row sq_head k sk_row sk_head v sv_row sv_head out so_row so_head lse cu_q cu_k seqs rows "
                 "keys heads kv_heads dim scale causal").split()
        values = dict.fromkeys(names, 0) | dict(heads=4, kv_heads=2, dim=64, scale=1.0) | fields
        return lib.kf_prefill_attention(native.PREFILL_ARGS.pack(*(values[n] for n in names)), None)

    assert prefill() == native.KF_OK
    assert prefill(kv_heads=3) == native.KF_ERR_INVALID_ARGUMENT
    assert prefill(kv_heads=0) == native.KF_ERR_INVALID_ARGUMENT
    assert prefill(dim=264) == native.KF_ERR_UNSUPPORTED
    assert prefill(rows=-1) == native.KF_ERR_INVALID_ARGUMENT
    assert prefill(rows=1 << 31) == native.KF_ERR_INVALID_ARGUMENT
    assert prefill(scale=math.inf) == native.KF_ERR_INVALID_ARGUMENT
    assert prefill(rows=5) == native.KF_ERR_INVALID_ARGUMENT and "null pointer" in native.last_error()


def test_cpu_tensors_are_refused():
    q, cu = torch.zeros(3, 2, 8), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA tensor"):
        prefill_attention(q, q, q, cu)
    with pytest.raises(ValueError, match="CUDA tensor"):
        tree_attention(q, q[None], q[None], cu[None], cu)
    with pytest.raises(ValueError, match="CUDA tensor"):
        rotary(q, q, cu, torch.zeros(4, 8))
    with pytest.raises(ValueError, match="CUDA tensor"):
        build_slots(cu, cu, cu[None], cu, block_size=16, max_tokens=4)


def test_rotary_table_scalings():
    plain = rotary_table(100, 16, device="cpu")
    assert plain.shape == (100, 16) and plain.dtype == torch.float32
    angle = 7 * 10000.0 ** (-torch.arange(0, 16, 2, dtype=torch.float64) / 16)
    assert torch.equal(plain[7], torch.cat([angle.cos(), angle.sin()]).float())
    # linear: position 4 p of a table stretched by 4 is position p of the plain one
    linear = rotary_table(400, 16, scaling="linear", factor=4.0, device="cpu")
    assert (linear[::4] - plain).abs().max() <= 2.0 ** -23
    # base: the fastest pair keeps its angles, the slowest turns a quarter as fast
    raised = rotary_table(400, 16, scaling="base", factor=4.0, device="cpu")
    assert torch.equal(raised[:100, 0], plain[:, 0])
    assert (raised[::4, 7] - plain[:, 7]).abs().max() <= 2.0 ** -22
    # parts: pairs with many turns keep theirs, those with few are divided
    parts = rotary_table(400, 16, scaling="parts", factor=4.0, original_positions=2000, low_turns=1.0, high_turns=32.0,
                         device="cpu")
    turns = 2000 * 10000.0 ** (-torch.arange(0, 16, 2) / 16) / (2 * math.pi)
    for i, n in enumerate(turns.tolist()):
        if n >= 32:
            assert (parts[:100, i] - plain[:, i]).abs().max() <= 2.0 ** -22
        elif n <= 1:
            assert (parts[::4, i] - plain[:, i]).abs().max() <= 2.0 ** -22
        else:
            assert (parts[:100, i] - plain[:, i]).abs().max() > 1e-3
    assert torch.equal(rotary_table(50, 16, scaling="parts", factor=1.0, original_positions=2000, device="cpu"),
                       plain[:50])


@pytest.mark.parametrize("kw,message", [
    (dict(rotary_dim=7), "even"), (dict(rotary_dim=0), "even"), (dict(scaling="ntk"), "scaling must be"),
    (dict(scaling="linear", factor=0.5), "factor"), (dict(scaling="parts", factor=2.0), "original_positions"),
    (dict(scaling="base", rotary_dim=2, factor=2.0), "two pairs"), (dict(max_positions=-1), "max_positions"),
])
def test_rotary_table_refusals(kw, message):
    with pytest.raises(ValueError, match=message):
        rotary_table(**(dict(max_positions=10, rotary_dim=16, device="cpu") | kw))


def test_a_workspace_off_its_alignment_is_refused_on_the_host():
    """Partial results are moved 16 bytes at a time: an address between would fault."""
    if torch.cuda.is_available():
        pytest.skip("the addresses are made up: only where nothing can be launched")
    lib = native.load()
    names = ("dtype q sq_row sq_head k_cache sk_page sk_head sk_slot v_cache sv_page sv_head sv_slot out so_row so_head lse "
             "block_table table_stride table_cols pages block_size context cu_q tree_mask mask_words seqs rows heads "
             "kv_heads dim scale workspace workspace_bytes").split()
    values = dict.fromkeys(names, 0) | dict(heads=4, kv_heads=2, dim=64, scale=1.0, block_size=16, rows=1, seqs=1, pages=1,
                                            table_cols=1, workspace_bytes=1 << 30)
    values |= dict.fromkeys(("q", "k_cache", "v_cache", "out", "block_table", "context"), 4096)  # never read here
    for off in (1, 8, 16, 128):
        packed = native.TREE_ARGS.pack(*((values | dict(workspace=4096 + off))[n] for n in names))
        assert lib.kf_tree_attention(packed, None) == native.KF_ERR_WORKSPACE
        assert "256-byte aligned" in native.last_error()


def test_overlaps_of_outputs_are_found():
    """Views of one buffer, against the elements that they really hold."""
    buf = torch.arange(4000)

    def held(t):
        return set(t.reshape(-1).tolist())

    gen = torch.Generator().manual_seed(0)
    for _ in range(3000):
        n, m, h, g, d = (int(x) for x in torch.randint(1, 6, (5,), generator=gen))
        strides = [int(x) for x in torch.randint(1, 40, (2,), generator=gen)]
        a, b = (buf.as_strided((rows, heads, d), (*strides, 1), int(torch.randint(0, 300, (1,), generator=gen)))
                for rows, heads in ((n, h), (m, g)))
        assert attention._overlap(a, b) == attention._overlap(b, a) == bool(held(a) & held(b))
        twice = len(held(a)) < a.numel()
        try:
            attention._check_output("out", a, {})
        except ValueError:
            continue  # it may refuse strides that interleave without meeting
        assert not twice
    qkv = torch.zeros(7, 12, 16)
    q, k, v, rest = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:8], qkv[:, 8:]
    attention._check_output("out", rest, {"q": q, "k": k, "v": v})
    attention._check_output("out", torch.zeros(4, 7, 16).transpose(0, 1), {"q": q})
    for out, other in ((q, q), (qkv[:, 1:5], q), (qkv[:, 7:11], v), (qkv.view(12, 7, 16)[:4].transpose(0, 1), q)):
        with pytest.raises(ValueError, match="shares memory with x"):
            attention._check_output("out", out, {"x": other})
    for out in (torch.zeros(1, 4, 16).expand(7, 4, 16), torch.zeros(7, 1, 16).expand(7, 4, 16)):
        with pytest.raises(ValueError, match="overlaps itself"):
            attention._check_output("out", out, {})


def test_c_entries_refuse_outputs_that_overlap():
    if torch.cuda.is_available():
        pytest.skip("the addresses are made up: only where nothing can be launched")
    lib = native.load()
    names = ("dtype q sq_row sq_head k sk_row sk_head v sv_row sv_head out so_row so_head lse cu_q cu_k seqs rows "
             "keys heads kv_heads dim scale causal").split()
    base = dict.fromkeys(names, 0) | dict(heads=4, kv_heads=2, dim=64, scale=1.0, rows=5, seqs=1, keys=5, so_row=256,
                                          so_head=64, q=4096, out=8192, k=4096, v=4096, cu_q=4096, cu_k=4096)
    for change, message in ((dict(out=4096), "must not be q"), (dict(so_row=0), "overlaps itself"),
                            (dict(so_head=0), "overlaps itself")):
        packed = native.PREFILL_ARGS.pack(*((base | change)[n] for n in names))
        assert lib.kf_prefill_attention(packed, None) == native.KF_ERR_INVALID_ARGUMENT
        assert message in native.last_error()


def test_counts_that_a_step_would_carry_past_32_bits_are_refused():
    """The kernels go through requests 32, rows 256 and keys 128 at a time, in 32 bits."""
    lib = native.load()
    names = ("dtype q sq_row sq_head k sk_row sk_head v sv_row sv_head out so_row so_head lse cu_q cu_k seqs rows "
             "keys heads kv_heads dim scale causal").split()
    base = dict.fromkeys(names, 0) | dict(heads=4, kv_heads=2, dim=64, scale=1.0)
    for name in ("rows", "keys", "seqs"):
        packed = native.PREFILL_ARGS.pack(*((base | {name: 0x7fffff01})[n] for n in names))
        assert lib.kf_prefill_attention(packed, None) == native.KF_ERR_INVALID_ARGUMENT, name
        assert "32 bits" in native.last_error()
    assert lib.kf_tree_attention_workspace_bytes(0, native.native_code(torch.bfloat16), 0x7fffff01, 1, 4, 2,
                                                 64) == -native.KF_ERR_INVALID_ARGUMENT

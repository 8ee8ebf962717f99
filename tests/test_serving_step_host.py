"""The host side of the operators around a decoding step, without a GPU: argument structs against the header, refusals of
the C entries and of the Python ones that need no device."""

from __future__ import annotations

import math
import re
from pathlib import Path

import pytest
import torch

from kernelo_b200.kernels.logits import adjust_logits
from kernelo_b200.kernels.paged import compact_pages, fork_requests, release_requests
from kernelo_b200.kernels.rotary import norm_rotary, norm_rotary_backward
from kernelo_b200.runtime import native

HEADER = (Path(__file__).resolve().parent.parent / "include" / "kernelo_b200.h").read_text()
STRUCTS = {"kf_norm_rotary_args": native.NORM_ROTARY_ARGS, "kf_norm_rotary_grad_args": native.NORM_ROTARY_GRAD_ARGS,
           "kf_logits_args": native.LOGITS_ARGS, "kf_fork_args": native.FORK_ARGS, "kf_release_args": native.RELEASE_ARGS,
           "kf_compact_args": native.COMPACT_ARGS}


def fields(name: str) -> dict[str, str]:
    """A struct's fields in order, those of nested structs in their place, each "q" or "d"."""
    body = re.search(r"typedef struct %s \{(.*?)\}" % name, HEADER, re.S).group(1)
    found = {}
    for line in filter(None, (re.sub(r"\s+", " ", part).strip() for part in body.split(";"))):
        kind, names = re.fullmatch(r"((?:const )?\w+(?: ?\*(?: const\*)?)?) ?(.*)", line).groups()
        if kind.startswith("kf_"):
            found |= fields(kind)
            continue
        assert "*" in kind or kind in ("int64_t", "double"), line
        for n in names.split(","):
            found[n.strip()] = "d" if kind == "double" else "q"
    return found


def packed(name: str, **values) -> bytes:
    known = fields(name)
    assert not set(values) - set(known)
    return STRUCTS[name].pack(*(values.get(n, 0) for n in known))


@pytest.mark.parametrize("name", STRUCTS)
def test_argument_structs_match_the_header(name):
    known = fields(name)
    letters = "".join(c * int(n or 1) for n, c in re.findall(r"(\d*)([a-z])", STRUCTS[name].format))
    assert letters == "".join(known.values()) and STRUCTS[name].size == 8 * len(known)


def refused(entry, name, status, message, **values):
    assert entry(packed(name, **values), None) == status, values
    assert message in native.last_error(), (values, native.last_error())


def test_c_entries_refuse_before_touching_a_device():
    lib = native.load()
    bad, unsupported = native.KF_ERR_INVALID_ARGUMENT, native.KF_ERR_UNSUPPORTED
    for entry in (lib.kf_norm_rotary, lib.kf_norm_rotary_grad, lib.kf_adjust_logits, lib.kf_fork, lib.kf_release, lib.kf_compact):
        assert entry(None, None) == bad
    heads = dict(tokens=3, heads=4, kv_heads=2, dim=64, eps=1e-6)
    for entry, name in ((lib.kf_norm_rotary, "kf_norm_rotary_args"), (lib.kf_norm_rotary_grad, "kf_norm_rotary_grad_args")):
        for change, message in ((dict(dtype=9), "dtype"), (dict(dim=-1), "negative"), (dict(rot=3), "even"),
                                (dict(heads=1 << 40), "32 bits"), (dict(eps=0.0), "eps"), (dict(eps=math.nan), "eps"),
                                (dict(eps=math.inf), "eps"), ({}, "null pointer")):
            refused(entry, name, bad, message, **(heads | change))
        refused(entry, name, unsupported, "at most 256", **(heads | dict(dim=257, tokens=0)))
        refused(entry, name, bad, "inverse", **(heads | dict(tokens=0, inverse=1)))
    assert lib.kf_norm_rotary(packed("kf_norm_rotary_args", **(heads | dict(tokens=0))), None) == native.KF_OK
    refused(lib.kf_norm_rotary_grad, "kf_norm_rotary_grad_args", bad, "null pointer", **(heads | dict(tokens=0)))
    refused(lib.kf_norm_rotary_grad, "kf_norm_rotary_grad_args", bad, "no cache", **(heads | dict(tokens=0, slots=4096)))
    assert lib.kf_norm_rotary_grad_workspace_bytes(0, -1, 1, 1, 1) == -bad

    rows = dict(rows=2, vocab=100)
    for change, message in ((dict(dtype=9), "dtype"), (dict(rows=-1), "negative"), (dict(rows=1 << 31), "32 bits"),
                            (dict(vocab=0x7fff0001), "32 bits"), (dict(token_cols=0x7fff0001), "32 bits"), ({}, "null pointer"),
                            (dict(logits=4096, out=4096, tokens=4096), "null pointer"),
                            (dict(logits=4096, out=4096, bias_tokens=4096), "null pointer"),
                            (dict(logits=4096, out=4096), "overlaps itself")):
        refused(lib.kf_adjust_logits, "kf_logits_args", bad, message, **(rows | change))
    assert lib.kf_adjust_logits(packed("kf_logits_args", rows=2), None) == native.KF_OK

    pool = dict(pages=4, heads=2, block_size=16, dim=8, rows=2, table_cols=3, block_table=4096, context=4096, holders=4096)
    for entry, name in ((lib.kf_fork, "kf_fork_args"), (lib.kf_compact, "kf_compact_args")):
        for change, message in ((dict(dtype=9), "dtype"), (dict(n_caches=-1), "negative"), (dict(block_size=0), "block_size"),
                                (dict(pages=1 << 31), "32 bits"), (dict(heads=1 << 20, dim=1 << 20), "32 bits"),
                                (dict(n_caches=1), "null pointer"), (dict(rows=(1 << 18) + 1), "rows"), (dict(rows=-1), "negative"),
                                (dict(block_table=0), "null pointer"), (dict(context=0), "null pointer"),
                                (dict(holders=0), "null pointer"), (dict(counts=0), "null pointer")):
            refused(entry, name, bad, message, **(pool | change))
    refused(lib.kf_compact, "kf_compact_args", unsupported, "at most 4194304", **(pool | dict(pages=(1 << 22) + 1)))
    fork = pool | dict(counts=4096, parents=4096, children=4096)
    for change, message in ((dict(pairs=-1), "negative"), (dict(pairs=1 << 30), "too many"), (dict(pairs=1, parents=0), "null pointer"),
                            (dict(n_free=1), "null pointer")):
        refused(lib.kf_fork, "kf_fork_args", bad, message, **(fork | change))
    table = dict(rows=2, table_cols=3, block_table=4096, context=4096, holders=4096, pages=4, block_size=16, n_freed=4096)
    for change, message in ((dict(pages=-1), "negative"), (dict(block_size=0), "block_size"), (dict(count=1), "null pointer"),
                            (dict(count=1 << 17, table_cols=1 << 13), "2^30"), (dict(n_freed=0), "null pointer")):
        refused(lib.kf_release, "kf_release_args", bad, message, **(table | change))


def test_cpu_tensors_are_refused():
    q, w, at = torch.zeros(3, 2, 8), torch.zeros(8), torch.zeros(3, dtype=torch.int32)
    for call in (lambda: norm_rotary(q, q, at, torch.zeros(4, 8), w, w),
                 lambda: norm_rotary_backward(q, q, q, q, at, torch.zeros(4, 8), w, w),
                 lambda: adjust_logits(q[0]),
                 lambda: fork_requests([q[None]], at[None], at[:1], at, at, at, at),
                 lambda: release_requests(at[None], at[:1], at, at, block_size=16),
                 lambda: compact_pages([q[None]], at[None], at[:1], at)):
        with pytest.raises(ValueError, match="CUDA tensor"):
            call()

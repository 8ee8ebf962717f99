"""Caches that forks and compactions refuse by their layout, without a GPU: the C entries' own checks."""

from __future__ import annotations

import array

import pytest

from kernelo_b200.runtime import native
from tests.test_serving_step_host import refused


@pytest.mark.parametrize("change", [dict(s_slot=7), dict(s_slot=0), dict(s_head=120), dict(s_page=255), dict(s_page=0),
                                    dict(s_head=8, s_slot=15)])
def test_caches_whose_slots_share_memory_are_refused(change):
    caches = array.array("Q", [0x10000000, 0x20000000])
    pool = dict(pages=4, heads=2, block_size=16, dim=8, s_page=256, s_head=128, s_slot=8, rows=2, table_cols=3, table_stride=3,
                block_table=4096, context=8192, holders=12288, n_caches=2, caches=caches.buffer_info()[0])
    lib = native.load()  # (counts is null: what passes the check is refused for that)
    for entry, name in ((lib.kf_fork, "kf_fork_args"), (lib.kf_compact, "kf_compact_args")):
        refused(entry, name, native.KF_ERR_INVALID_ARGUMENT, "null pointer", **pool)
        refused(entry, name, native.KF_ERR_INVALID_ARGUMENT, "caches overlap themselves", **(pool | change))
        refused(entry, name, native.KF_ERR_INVALID_ARGUMENT, "null pointer", **(pool | dict(s_head=8, s_slot=16)))

"""What a serving block's geometry refuses before anything is made of it."""

from __future__ import annotations

import pytest

from kernelo_b200.integration import ServingConfig


def test_head_norms_of_heads_that_are_too_wide_are_refused():
    wide = dict(hidden=1032, heads=4, kv_heads=2)
    with pytest.raises(ValueError, match="at most 256 elements, got 258"):
        ServingConfig(**wide, qk_norm=True)
    assert ServingConfig(**wide).head_dim == 258
    assert ServingConfig(hidden=1024, heads=4, kv_heads=2, qk_norm=True).head_dim == 256

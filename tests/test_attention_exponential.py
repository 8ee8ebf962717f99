"""The polynomial that stands in for part of the exponentials of prompt attention, in
fp32 arithmetic on the host with the kernel's own constants."""

from __future__ import annotations

import re
from pathlib import Path

import numpy as np

SOURCE = Path(__file__).resolve().parent.parent / "kernelo_b200" / "csrc" / "attention_softmax.cuh"
f32 = np.float32


def exponential(x):
    """2^x as the kernel computes it: fused multiply-adds in 64 bits, rounded to 32."""
    body = re.search(r"ex2_poly2\(float2 v\) \{(.*?)\n\}", SOURCE.read_text(), re.S).group(1)
    least = f32(re.search(r"fmaxf\(v\.x, (-?[0-9.]+)f\)", body).group(1))
    magic, _, *terms = (f32(c) for c in re.findall(r"f2_splat\((-?[0-9.]+)f\)", body))
    assert len(terms) == 5
    x = np.maximum(x.astype(f32), least)
    t = (x + magic).astype(f32)
    f = (x + (magic - t)).astype(f32)
    r = np.full_like(f, terms[0])
    for c in terms[1:]:
        r = (r.astype(np.float64) * f + np.float64(c)).astype(f32)
    bits = r.view(np.int32).astype(np.int64) + (t.view(np.int32).astype(np.int64) << 23)
    return (bits & 0xFFFFFFFF).astype(np.uint32).view(f32)


def test_relative_error():
    """The stated error, over all that a weight can be: 2^-126 to the 2^8 that a maximum may be left behind."""
    x = np.linspace(-126, 8, 2_000_003).astype(f32)
    got = exponential(x).astype(np.float64)
    assert np.abs(got / np.exp2(x.astype(np.float64)) - 1).max() <= 2.9e-6


def test_masked_keys_weigh_exactly_nothing():
    assert (exponential(np.array([-127, -128, -1e30, -np.inf])).view(np.int32) == 0).all()


def test_below_the_normal_numbers():
    """Every number from -127 to -126: no sign, nothing above the least normal number."""
    x = -np.arange(f32(126).view(np.int32), f32(127).view(np.int32) + 1).astype(np.int32).view(f32)
    bits = exponential(x).view(np.int32)
    assert (bits >= 0).all() and (bits <= f32(2.0 ** -126).view(np.int32)).all()

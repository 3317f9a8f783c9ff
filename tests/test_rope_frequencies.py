"""Rotary frequencies of stretched contexts, pair by pair, against the rule stated apart.

YaRN keeps the pairs that turn more than 32 times in the trained length, divides those that turn
less than once by the factor, and blends the two linearly over the pair index in between. The ramp's
ends are the pair indexes where the turns are 32 and 1, rounded outward; the slow end may lie past
the last pair, which then turns more than once and keeps a part of its frequency.
"""

from __future__ import annotations

import math

import numpy as np
import pytest

from plastic_infer_b200 import kernels


def yarn(dim, base, factor, trained):
    """Frequencies by the turns of each pair, the ramp's ends found by search over the pairs."""
    def turns(j):
        return trained * base ** (-2.0 * j / dim) / (2 * math.pi)

    low = max((j for j in range(dim) if turns(j) >= 32.0), default=0)
    high = min((j for j in range(dim) if turns(j) <= 1.0), default=dim - 1)
    j = np.arange(dim // 2)
    w = np.clip((j - low) / max(high - low, 1e-3), 0, 1)
    f = base ** (-2.0 * j / dim)
    return (1 - w) * f + w * f / factor, np.array([turns(x) for x in j])


@pytest.mark.parametrize("dim,base,factor,trained", [
    (128, 1e4, 4.0, 4096), (128, 1e4, 4.0, 65536), (128, 1e4, 4.0, 131072), (64, 1e4, 8.0, 131072),
    (64, 1e4, 2.0, 1 << 20), (128, 1e6, 4.0, 32768), (128, 5e5, 16.0, 131072), (32, 100.0, 4.0, 4096),
])
def test_yarn_every_pair(dim, base, factor, trained):
    want, turns = yarn(dim, base, factor, trained)
    got, scale = kernels.rope_frequencies(dim, base, "yarn", factor, trained)
    # fp32 values of a 64-bit computation: half a step, and as much again for the powers
    np.testing.assert_allclose(got.double().numpy(), want, rtol=2.0 ** -23)
    assert scale == pytest.approx(0.1 * math.log(factor) + 1)
    plain = base ** (-2.0 * np.arange(dim // 2) / dim)
    slow = turns < 1
    np.testing.assert_allclose(got.double().numpy()[slow], plain[slow] / factor, rtol=2.0 ** -23)
    if not slow.any():  # the slowest pair is not stretched by the whole factor
        assert float(got[-1]) > plain[-1] / factor * 1.05

"""The YaRN rotary frequencies, pair by pair, against the published rule written out apart: the ramp over the pair number
from floor(pair that turns beta_fast times over the original context), at least 0, to ceil(pair that turns beta_slow times), at
most rotary_dim - 1. The second bound is beyond the last pair, rotary_dim / 2 - 1: where that pair still turns
more than beta_slow times the ramp ends behind it.
"""
import math

import pytest

from mi50_vllm_lab_amd import rotary


def published(dim, base, factor, original, fast=32.0, slow=1.0):
    def number(turns):
        return dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))

    low, high = max(math.floor(number(fast)), 0), min(math.ceil(number(slow)), dim - 1)
    out = []
    for i in range(dim // 2):
        f = base ** (-2 * i / dim)
        ramp = min(max((i - low) / (high - low), 0.0), 1.0)
        out.append(f / factor * ramp + f * (1 - ramp))
    return out


@pytest.mark.parametrize("dim,base,factor,original,kw", [
    (128, 1e4, 4, 131072, {}),                 # the last pair turns 2.4 times
    (64, 1e4, 4, 65536, {}),
    (64, 1e4, 8, 131072, {}),
    (128, 1e4, 8, 65536, {}),
    (128, 1e4, 16, 4096, {}),                  # the ramp ends before the last pair
    (256, 1e6, 4, 262144, {}),
    (64, 5e5, 32, 8192, {"beta_fast": 16.0, "beta_slow": 2.0}),
    (32, 1e4, 2, 100, {}),                     # no pair turns beta_fast times
    (8, 1e4, 2, 1 << 20, {}),
])
def test_every_pair(dim, base, factor, original, kw):
    got, _ = rotary.rotary_frequencies(dim, base, {"type": "yarn", "factor": factor, "original_max_position": original, **kw})
    want = published(dim, base, factor, original, kw.get("beta_fast", 32.0), kw.get("beta_slow", 1.0))
    assert max(abs(g / w - 1) for g, w in zip(got.tolist(), want)) < 1e-12


def test_a_last_pair_that_turns_often_is_not_divided_fully():
    for dim, original in ((128, 131072), (64, 65536), (64, 131072)):
        plain, _ = rotary.rotary_frequencies(dim, 1e4)
        got, _ = rotary.rotary_frequencies(dim, 1e4, {"type": "yarn", "factor": 8, "original_max_position": original})
        assert float(plain[-1]) * original / (2 * math.pi) > 1.0 and float(got[-1]) > float(plain[-1]) / 8 * 1.5

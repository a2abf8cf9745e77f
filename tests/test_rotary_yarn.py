"""The "yarn" frequencies of macai_b200.rotary against the published method, on the CPU: pair i of dim / 2 keeps its speed
below the ramp, is slowed by `factor` past it, and in between the two are mixed by ramp((i - low) / (high - low)), where
low and high are the pairs that turn `fast` and `slow` times within the original length, low = max(floor, 0) and
high = min(ceil, dim - 1): a ramp that ends past the last pair keeps its slope."""
import math

import pytest
import torch


def _published(dim, base, factor, length, fast=32.0, slow=1.0):
    at = [dim * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(base)) for turns in (fast, slow)]
    low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), dim - 1)
    out = []
    for i in range(dim // 2):
        speed = base ** (-2 * i / dim)
        part = min(max((i - low) / max(high - low, 1e-3), 0.0), 1.0)
        out.append(speed * (1 - part) + speed / factor * part)
    return torch.tensor(out, dtype=torch.float64)


@pytest.mark.parametrize("dim,base,factor,length", [
    (64, 1e4, 4.0, 4096), (64, 1e4, 4.0, 32768), (64, 1e4, 4.0, 65536), (64, 1e4, 4.0, 131072), (128, 1e4, 8.0, 131072),
    (128, 1e6, 4.0, 32768), (32, 1e4, 2.0, 1 << 20), (8, 1e4, 16.0, 1 << 18)])
def test_yarn_is_the_published_ramp(dim, base, factor, length):
    """Equal to the rounding of a few float64 operations."""
    from macai_b200.rotary import rotary_frequencies
    got, _ = rotary_frequencies(dim, base, {"type": "yarn", "factor": factor, "original_length": length})
    assert torch.allclose(got, _published(dim, base, factor, length), rtol=1e-12, atol=0)


def test_a_pair_that_turns_more_than_once_is_not_slowed_in_full():
    from macai_b200.rotary import rotary_frequencies
    for length in (65536, 131072, 1 << 20):
        plain, _ = rotary_frequencies(64)
        got, _ = rotary_frequencies(64, scaling={"type": "yarn", "factor": 4.0, "original_length": length})
        more = plain * length / (2 * math.pi) > 1.1
        assert (got[more] > plain[more] / 4 * (1 + 1e-9)).all(), length

"""Stretched rotary frequencies, every pair against the number of times it turns (CPU)."""
import math

import pytest
import torch

from custom_ops_b200 import rotary_frequencies


def turns_of(index, rot, base, length):
    """Turns of the pair with this index, which may lie outside the head's, within `length` positions."""
    return length * base ** (-2.0 * index / rot) / (2.0 * math.pi)


@pytest.mark.parametrize("rot,base,length", [
    (128, 10000.0, 4096),                  # both ends of the ramp among the pairs
    (128, 10000.0, 131072), (64, 10000.0, 65536), (64, 10000.0, 131072),     # the slowest pair turns more than `slow` times
    (128, 10000.0, 40), (20, 500.0, 100),  # the fastest turns less than `fast` times
    (64, 10000.0, 4),                      # the fastest turns less than `slow` times
    (64, 100.0, 1 << 20),                  # the slowest turns more than `fast` times
    (2, 10000.0, 64), (2, 10000.0, 4), (2, 10000.0, 1 << 20),
])
@pytest.mark.parametrize("fast,slow", [(32.0, 1.0), (9.0, 8.5)])
def test_by_parts_goes_by_the_turns_of_each_pair(rot, base, length, fast, slow):
    factor = 4.0
    f, _ = rotary_frequencies(rot, base, device="cpu")
    g, mscale = rotary_frequencies(rot, base, scaling="by_parts", factor=factor, original_length=length, fast=fast, slow=slow,
                                   device="cpu")
    assert g.dtype == torch.float64 and abs(mscale - (0.1 * math.log(factor) + 1.0)) < 1e-15
    # the last index that still turns `fast` times and the first that turns no more than `slow` times
    indices = range(-8 * rot, 8 * rot)
    lo = max(k for k in indices if turns_of(k, rot, base, length) >= fast)
    hi = min(k for k in indices if turns_of(k, rot, base, length) <= slow)
    assert lo < hi
    for i in range(rot // 2):
        turns, ratio = turns_of(i, rot, base, length), (g[i] / f[i]).item()
        if turns >= fast:
            assert ratio == 1.0, i
        elif turns <= slow:
            assert abs(ratio * factor - 1.0) < 1e-12, i
        else:
            assert 1.0 / factor < ratio < 1.0, i
        weight = min(max((i - lo) / (hi - lo), 0.0), 1.0)
        assert abs(ratio - (1.0 - weight + weight / factor)) < 1e-12, i


def test_by_parts_of_a_slowest_pair_within_the_ramp():
    """By hand: 64 pairs of base 10000 over 131072 positions.  Index of 32 turns: 64 ln(131072 / (64 pi)) / ln 10000 =
    45.03, of one turn 69.11; the ramp goes from 45 to 70, and the last pair, 63, has done 18 of its 25 steps."""
    f, _ = rotary_frequencies(128, 10000.0, device="cpu")
    g, _ = rotary_frequencies(128, 10000.0, scaling="by_parts", factor=4.0, original_length=131072, device="cpu")
    assert abs((g[63] / f[63]).item() - (1.0 - 0.75 * 18 / 25)) < 1e-12
    assert torch.equal(g[:46], f[:46])

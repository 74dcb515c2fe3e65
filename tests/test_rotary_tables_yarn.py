"""The ramp of rotary.rotary_tables(scaling="yarn") against its formula pair by pair, on the CPU."""
import math

import pytest
import torch


def published(dim, theta, factor, trained, fast, slow):
    """The angles of position 1, one pair at a time: within the trained positions pair x turns
    trained theta^(-2x/dim) / (2 pi) times, so n times at x = dim log(trained / (2 pi n)) / (2 log theta); the share of the
    divided angle rises linearly from the pair below the one with `fast` turns (at least 0) to the one above that with
    `slow` turns (at most dim - 1)."""
    x = lambda n: dim * math.log(trained / (2 * math.pi * n)) / (2 * math.log(theta))
    first, last = max(math.floor(x(fast)), 0), min(math.ceil(x(slow)), dim - 1)
    rates = []
    for pair in range(dim // 2):
        rate = theta ** (-2 * pair / dim)
        share = min(max((pair - first) / (last - first), 0.0), 1.0) if last > first else float(pair > first)
        rates.append(rate * (1 - share) + rate / factor * share)
    return rates


@pytest.mark.parametrize("dim,theta,trained,fast,slow", [
    (128, 1e4, 131072, 32.0, 1.0), (64, 1e4, 131072, 32.0, 1.0), (64, 1e4, 47000, 32.0, 1.0), (128, 1e4, 4096, 32.0, 1.0),
    (64, 1e4, 2048, 32.0, 1.0), (64, 1e4, 150, 32.0, 1.0), (16, 100.0, 10**6, 32.0, 1.0), (16, 100.0, 10**9, 32.0, 1.0),
    (96, 5e5, 8192, 16.0, 2.0), (64, 1e4, 2048, 4.0, 4.0)])
def test_every_pair(dim, theta, trained, fast, slow):
    from mathbrain.rotary import rotary_tables
    for factor in (1.0, 4.0, 40.0):
        cos, sin = rotary_tables(dim, 2, theta, "yarn", factor, trained, fast, slow)
        size = 0.1 * math.log(factor) + 1
        for pair, rate in enumerate(published(dim, theta, factor, trained, fast, slow)):
            # the tables round to fp32, 2^-24 relative of values up to `size` (at most 1.37)
            assert abs(float(cos[1, pair]) - size * math.cos(rate)) < 2.0**-23, (factor, pair)
            assert abs(float(sin[1, pair]) - size * math.sin(rate)) <= 2.0**-23 * size * math.sin(rate) + 1e-12, (factor, pair)


def test_a_slowest_pair_that_turns_is_divided_in_part():
    from mathbrain.rotary import rotary_tables
    cos, sin = rotary_tables(128, 2, 1e4, "yarn", 4.0, 131072)
    plain = 1e4 ** (-126 / 128)
    ratio = math.atan2(float(sin[1, 63]), float(cos[1, 63])) / plain
    assert 131072 * plain / (2 * math.pi) > 2.4 and abs(ratio - 0.46) < 0.005


def test_all_pairs_slow():
    """So few trained positions that even the fastest pair turns less than once: all are divided."""
    from mathbrain.rotary import rotary_tables
    cos, sin = rotary_tables(8, 2, 100.0, "yarn", 2.0, trained=4)
    want = 100.0 ** (-torch.arange(0, 8, 2, dtype=torch.float64) / 8) / 2
    assert (torch.atan2(sin[1].double(), cos[1].double()) - want).abs().max() < 1e-6


@pytest.mark.parametrize("bad", [dict(theta=1.0), dict(theta=0.0), dict(theta=-5.0), dict(theta=math.nan), dict(fast=1.0, slow=2.0),
                                 dict(slow=0.0), dict(fast=math.inf)])
def test_refusals(bad):
    from mathbrain.rotary import rotary_tables
    with pytest.raises(ValueError, match="theta"):
        rotary_tables(**(dict(dim=64, positions=8, scaling="yarn", factor=2.0, trained=64) | bad))

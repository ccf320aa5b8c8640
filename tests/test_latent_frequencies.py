"""Frequencies of stretched contexts against their definition, for trained lengths at which the slowest pair turns less and more than once."""

import math

import pytest
import torch

from ascendflow_b200 import latent


@pytest.mark.parametrize("dims,base,length,factor,fast,slow", [
    (64, 10000.0, 4096, 8.0, 32.0, 1.0), (64, 10000.0, 32768, 4.0, 32.0, 1.0), (64, 10000.0, 65536, 16.0, 32.0, 1.0), (64, 10000.0, 131072, 4.0, 32.0, 1.0),
    (128, 10000.0, 1 << 20, 2.0, 32.0, 1.0), (64, 500000.0, 8192, 8.0, 4.0, 1.0), (16, 100.0, 4096, 40.0, 64.0, 2.0), (64, 10.0, 65536, 8.0, 32.0, 1.0),
])
def test_yarn(dims, base, length, factor, fast, slow):
    """Pair x turns length * base ** (-2 x / dims) / (2 pi) times. From the whole pair below the one that turns `fast` times to the whole pair above the one that turns `slow`
    times, wherever those lie, the share that is divided by the factor goes from 0 to 1. (Each frequency: three roundings to 2^-53.)"""
    half = dims // 2

    def bisect(turns):  # where a pair would turn so often
        low, high = -10.0 * half, 10.0 * half
        for _ in range(200):
            middle = (low + high) / 2
            low, high = (middle, high) if length * base ** (-middle / half) / (2 * math.pi) > turns else (low, middle)
        return low

    first, last = max(math.floor(bisect(fast)), 0), min(math.ceil(bisect(slow)), dims - 1)
    found = latent.rotary_frequencies(dims, base=base, scaling="yarn", factor=factor, original_length=length, beta_fast=fast, beta_slow=slow, device="cpu")
    for pair in range(half):
        plain = base ** (-pair / half)
        share = min(max((pair - first) / (last - first), 0.0), 1.0) if last > first else 0.0
        expected = plain * (1 - share) + plain / factor * share
        assert abs(found[pair].item() / expected - 1) < 1e-14, pair
        turns = length * plain / (2 * math.pi)
        if turns > fast * 1.000001:
            assert found[pair].item() == pytest.approx(plain, rel=1e-14)
        if turns < slow * 0.999999:
            assert found[pair].item() == pytest.approx(plain / factor, rel=1e-14)


def test_yarn_where_the_slowest_pair_still_turns():
    """A trained length of 65536: the last pair of 64 features turns 1.39 times, and is on the ramp."""
    plain = latent.rotary_frequencies(64, device="cpu")
    assert 65536 * plain[-1].item() / (2 * math.pi) > 1.39
    found = latent.rotary_frequencies(64, scaling="yarn", factor=16.0, original_length=65536, device="cpu")
    assert torch.allclose(found[-1] / plain[-1], torch.tensor(0.207, dtype=torch.float64), atol=1e-3)

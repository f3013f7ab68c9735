"""Stretched rotary frequencies against the statement of the ramp, pair by pair in Python's numbers."""
import math

import pytest
import torch

import channelestimationtransformer_amd as cet


def yarn(dim, base, factor, length, turns):
    """Rate of each pair: kept up to the last pair that turns more than turns[0] times in `length`, divided by `factor` from
    the first that turns less than turns[1] times on, and a straight line in the pair's number between those two."""
    at = [dim * math.log(length / (2 * math.pi * n)) / (2 * math.log(base)) for n in turns]  # pairs that turn just so often
    low, high = max(math.floor(at[0]), 0), math.ceil(at[1])
    out = []
    for j in range(dim // 2):
        rate = base ** (-2.0 * j / dim)
        share = 0.0 if j <= low and rate * length / (2 * math.pi) > turns[1] else 1.0 if j >= high else (j - low) / (high - low)
        out.append(rate * (1 - share) + rate / factor * share)
    return out


# 1.0: the rate kept, 0.125: divided by 8; the values between from the formula by hand
@pytest.mark.parametrize("dim, length, pair, share", [(4, 4096, 1, 0.5625), (6, 4096, 2, 5 / 12), (8, 8192, 3, 5 / 12), (64, 65536, 31, 0.260),
                                                      (128, 131072, 63, 0.370), (64, 4096, 0, 1.0), (64, 4096, 31, 0.125), (2, 4, 0, 0.125)])
def test_single_pairs(dim, length, pair, share):
    f, _ = cet.rotary_frequencies(dim, scaling="yarn", factor=8.0, original_length=length, device="cpu")
    assert abs(float(f[pair]) * 10000.0 ** (2 * pair / dim) - share) < 6e-4


@pytest.mark.parametrize("dim", [2, 4, 6, 8, 20, 64, 128, 256])
@pytest.mark.parametrize("length", [5, 64, 4096, 8192, 65536, 131072, 1 << 20])
@pytest.mark.parametrize("base, turns", [(10000.0, (32.0, 1.0)), (500000.0, (32.0, 1.0)), (10000.0, (8.0, 2.0))])
def test_every_pair(dim, length, base, turns):
    f, gain = cet.rotary_frequencies(dim, base=base, scaling="yarn", factor=8.0, original_length=length, turns=turns, device="cpu")
    want = torch.tensor(yarn(dim, base, 8.0, length, turns), dtype=torch.float64)
    assert torch.allclose(f, want, rtol=1e-12, atol=0.0)
    plain, _ = cet.rotary_frequencies(dim, base=base, device="cpu")
    n = plain * length / (2 * math.pi)
    assert torch.allclose(f[n < turns[1]], plain[n < turns[1]] / 8, rtol=1e-12)
    assert torch.equal(f[n > turns[0]][:-1], plain[n > turns[0]][:-1])  # (the last of them may be the ramp's first)
    assert abs(gain - (0.1 * math.log(8.0) + 1.0)) < 1e-12

"""rope_inv_freq over original lengths, against its own rule by the number of turns."""
import math

import pytest
import torch

import focal_b200 as F


@pytest.mark.parametrize("rot", [16, 64, 96, 128])
@pytest.mark.parametrize("base", [10000.0, 500000.0])
@pytest.mark.parametrize("original", [512, 4096, 32768, 62000, 63000, 131072, 1048576, 1 << 24])
def test_yarn_divides_only_slow_pairs(rot, base, original):
    """A pair that turns more than `low` times over the original length is not divided in full, one
    that turns more than `high` times is kept, one that turns less than `low` times is divided.
    (0.1 % beside the borders, where the logarithm's rounding decides.)"""
    factor = 8.0
    plain, _ = F.rope_inv_freq(rot, base=base, device="cpu")
    f, _ = F.rope_inv_freq(rot, base=base, scaling="yarn", factor=factor, original_max_position=original, device="cpu")
    turns = original * plain / (2 * math.pi)
    assert torch.all(f[turns > 1.001] > plain[turns > 1.001] / factor * (1 + 1e-9))
    assert torch.allclose(f[turns > 32.04], plain[turns > 32.04], rtol=1e-14)
    assert torch.allclose(f[turns < 0.999], plain[turns < 0.999] / factor, rtol=1e-14)


def test_yarn_keeps_everything_that_turns_often():
    """An original length over which the slowest pair turns more than `high` times: nothing is divided."""
    plain, _ = F.rope_inv_freq(64, device="cpu")
    f, m = F.rope_inv_freq(64, scaling="yarn", factor=4.0, original_max_position=1 << 24, device="cpu")
    assert torch.equal(f, plain) and m == 0.1 * math.log(4.0) + 1.0

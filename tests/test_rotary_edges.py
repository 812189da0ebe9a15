"""Edges of the rotary frequencies, beside tests/test_rotary.py."""

import math

import pytest
import torch

import memt_b200 as M


@pytest.mark.parametrize("trained,slow", [(4, 1.0), (6, 1.0), (100, 20.0), (4096, 700.0)])
def test_yarn_divides_every_pair_that_turns_slowly(trained, slow):
    """No pair makes slow_turns turns over the trained context: all are divided by the factor."""
    assert trained / (2 * math.pi) < slow  # the fastest pair turns by one radian a position
    plain, _ = M.rotary_frequencies(64, device="cpu")
    inv, _ = M.rotary_frequencies(64, scaling="yarn", factor=8.0, trained_tokens=trained, slow_turns=slow,
                                  fast_turns=2 * slow, device="cpu")
    assert torch.equal(inv, plain / 8.0)


@pytest.mark.parametrize("trained", [1, 7, 40, 300, 4096, 10 ** 6])
@pytest.mark.parametrize("dim,slow,fast", [(2, 1.0, 32.0), (64, 1.0, 32.0), (128, 0.5, 0.5), (256, 3.0, 17.0)])
def test_yarn_keeps_fast_and_divides_slow_pairs(dim, slow, fast, trained):
    plain, _ = M.rotary_frequencies(dim, device="cpu")
    inv, att = M.rotary_frequencies(dim, scaling="yarn", factor=4.0, trained_tokens=trained, slow_turns=slow,
                                    fast_turns=fast, device="cpu")
    turns = trained * plain / (2 * math.pi)
    keep, divided = turns > fast * (1 + 1e-9), turns < slow * (1 - 1e-9)
    assert torch.equal(inv[keep], plain[keep]) and torch.equal(inv[divided], plain[divided] / 4.0)
    assert bool(((inv <= plain) & (inv >= plain / 4.0 * (1 - 1e-15))).all()) and math.isclose(att, 0.1 * math.log(4) + 1)


@pytest.mark.parametrize("over", [dict(slow_turns=0.0), dict(slow_turns=-1.0), dict(slow_turns=33.0),
                                  dict(fast_turns=0.5), dict(trained_tokens=0)])
def test_yarn_refuses(over):
    with pytest.raises(ValueError):
        M.rotary_frequencies(64, **{"scaling": "yarn", "factor": 2.0, "trained_tokens": 512, "device": "cpu", **over})

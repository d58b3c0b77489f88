"""Scaled rotary frequencies against the published definition of yarn, written out here from the formulas, and what a configuration may hold."""

import math

import pytest

from himuon_b200 import ops


def _freqs(rotary_dim, theta, scaling):
    f = ops.RotaryFrequencies(rotary_dim, theta, scaling, device="cpu")
    return f.frequencies, f.factor


def _yarn(d, theta, s, beta_fast=32.0, beta_slow=1.0, truncate=True):
    """Angles at position 1: a pair that turns more than beta_fast times within the original length keeps its frequency, one that turns less than
    beta_slow times has it divided, and between the pairs where that is so there is a ramp."""
    length = s["original_max_position_embeddings"]
    # theta^(-2 i / d) * length / 2 pi turns: as many as beta at i = d ln(length / (2 pi beta)) / (2 ln theta)
    first, last = (d / 2 * (math.log(length) - math.log(2 * math.pi) - math.log(beta)) / math.log(theta) for beta in (beta_fast, beta_slow))
    if truncate:
        first, last = math.floor(first), math.ceil(last)
    first, last = max(first, 0), min(last, d - 1)
    out = []
    for i in range(d // 2):
        w = math.exp(-2 * i / d * math.log(theta))
        divided = min(1.0, max(0.0, (i - first) / (last - first)))
        out.append((1 - divided) * w + divided * w / s["factor"])
    return out


def _near(got, want):
    return len(got) == len(want) and all(math.isclose(a, b, rel_tol=1e-12) for a, b in zip(got, want))


YARN = {"rope_type": "yarn", "factor": 32.0, "original_max_position_embeddings": 4096}


@pytest.mark.parametrize("d,theta", [(64, 150000.0), (128, 10000.0), (64, 1000000.0), (20, 500.0)])
def test_yarn_with_and_without_whole_pairs(d, theta):
    """``truncate`` says whether the ramp starts and ends at whole pairs."""
    for truncate in (None, True, False):
        s = dict(YARN) if truncate is None else {**YARN, "truncate": truncate}
        assert _near(_freqs(d, theta, s)[0], _yarn(d, theta, s, truncate=truncate is not False)), truncate
    s = {**YARN, "beta_fast": 8.0, "beta_slow": 2.5, "truncate": False}
    assert _near(_freqs(d, theta, s)[0], _yarn(d, theta, s, 8.0, 2.5, False))
    for wrong in (1, 0.0, "false"):
        with pytest.raises(RuntimeError, match="truncate"):
            _freqs(d, theta, {**YARN, "truncate": wrong})

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


def test_yarn_factor_of_cosine_and_sine():
    """0.1 k ln factor + 1 for k = 1, or the quotient of two of them, or as given; 1 where nothing is stretched."""
    def m(k, factor):
        return 0.1 * k * math.log(factor) + 1.0

    for factor in (40.0, 1.5):
        s = {**YARN, "factor": factor}
        assert math.isclose(_freqs(64, 1e4, s)[1], m(1.0, factor), rel_tol=1e-15)
        for k, all_dim in ((1.0, 1.0), (0.707, 0.707), (1.0, 0.8), (0.4, 1.2)):
            got, scale = _freqs(64, 1e4, {**s, "mscale": k, "mscale_all_dim": all_dim})
            assert math.isclose(scale, m(k, factor) / m(all_dim, factor), rel_tol=1e-15) and got == _freqs(64, 1e4, s)[0]
        assert _freqs(64, 1e4, {**s, "mscale": 1.0, "mscale_all_dim": 1.0})[1] == 1.0
        assert _freqs(64, 1e4, {**s, "mscale": 1.0, "mscale_all_dim": 2.0, "attention_factor": 1.25})[1] == 1.25
        # one of them alone means different things to different readers
        for alone in ({"mscale": 1.0}, {"mscale_all_dim": 1.0}, {"mscale": 0.707, "mscale_all_dim": None}, {"mscale": 0.707, "mscale_all_dim": 0}):
            with pytest.raises(RuntimeError, match="mscale"):
                _freqs(64, 1e4, {**s, **alone})
    assert _freqs(64, 1e4, {**YARN, "factor": 0.5, "mscale": 1.0, "mscale_all_dim": 0.5})[1] == 1.0 == _freqs(64, 1e4, {**YARN, "factor": 1.0})[1]


def test_keys_without_a_value_are_not_there():
    absent = dict.fromkeys(("beta_fast", "beta_slow", "truncate", "attention_factor", "mscale", "mscale_all_dim"))
    assert _freqs(64, 1e4, {**YARN, **absent}) == _freqs(64, 1e4, YARN)
    assert _freqs(64, 1e4, {"rope_type": None, "type": "linear", "factor": 4.0}) == _freqs(64, 1e4, {"rope_type": "linear", "factor": 4.0})
    with pytest.raises(RuntimeError, match="needs factor"):
        _freqs(64, 1e4, {"rope_type": "linear", "factor": None})


LLAMA3 = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_max_position_embeddings": 8192}


def test_keys_that_are_not_known_are_refused():
    """Whatever a form does not take may change its frequencies."""
    linear, ntk, default = {"rope_type": "linear", "factor": 4.0}, {"rope_type": "ntk", "factor": 4.0}, {"rope_type": "default"}
    for s in (linear, ntk, default, LLAMA3):
        for key, value in (("beta_fast", 16.0), ("mscale", 1.0), ("truncate", False), ("attention_factor", 1.0)):
            with pytest.raises(RuntimeError, match=f"RotaryFrequencies: .*{key}"):
                _freqs(64, 1e4, {**s, key: value})
    for s in (linear, ntk, default, YARN, LLAMA3):
        for key, value in (("partial_rotary_factor", 0.5), ("mrope_section", [16, 24, 24]), ("short_factor", [1.0] * 32), ("Factor", 2.0), (5, 2.0)):
            with pytest.raises(RuntimeError, match=f"RotaryFrequencies: .*{key}"):
                _freqs(64, 1e4, {**s, key: value})
    for s in (default, YARN):
        with pytest.raises(RuntimeError, match="low_freq_factor"):
            _freqs(64, 1e4, {**s, "low_freq_factor": 1.0})
    with pytest.raises(RuntimeError, match="factor"):
        _freqs(64, 1e4, {**default, "factor": 4.0})


def test_keys_that_say_the_same_twice_have_to_agree():
    """Configurations have the form under both of its names, and the base beside the scaling."""
    for s in (YARN, LLAMA3, {"rope_type": "default"}):
        want = _freqs(64, 1e4, s)
        assert _freqs(64, 1e4, {**s, "type": s["rope_type"], "rope_theta": 10000}) == want
        with pytest.raises(RuntimeError, match="rope_type"):
            _freqs(64, 1e4, {**s, "type": "mrope"})
        with pytest.raises(RuntimeError, match="rope_theta"):
            _freqs(64, 1e4, {**s, "rope_theta": 500000.0})
    # lengths have no part in these
    assert _freqs(64, 1e4, {"rope_type": "linear", "factor": 4.0, "original_max_position_embeddings": 4096}) == _freqs(64, 1e4, {"rope_type": "linear", "factor": 4.0})

"""Keys of a scaling that change frequencies or scale, against the formulas."""
import math

import numpy as np
import pytest

from ncmorph_amd import decoder

YARN = dict(type="yarn", factor=8.0, original_max_position_embeddings=4096)


def test_yarn_of_two_scales():
    """mscale and mscale_all_dim: sines and cosines times the ratio of what each
    makes of the factor, 0.1 m ln factor + 1; attention_factor goes before them."""
    def scale(**k):
        return decoder.rope_frequencies(64, 1e4, dict(YARN, **k))[1]

    of = lambda m: 0.1 * m * math.log(8.0) + 1.0  # noqa: E731
    assert scale(mscale=1.0, mscale_all_dim=1.0) == 1.0
    assert abs(scale(mscale=0.707, mscale_all_dim=1.0) - of(0.707) / of(1.0)) < 1e-12
    assert scale(mscale=2.0, mscale_all_dim=1.0, attention_factor=1.5) == 1.5
    assert scale(mscale=2.0, mscale_all_dim=1.0, factor=1.0) == 1.0
    assert scale(mscale=None, mscale_all_dim=None) == of(1.0)
    for one in (dict(mscale=1.0), dict(mscale_all_dim=1.0)):   # of which the other is not known
        with pytest.raises(ValueError):
            scale(**one)
    assert scale(mscale=1.0, attention_factor=1.5) == 1.5


def test_yarn_without_whole_pairs():
    """truncate false: the ramp between the very pairs, not the whole ones."""
    whole, _ = decoder.rope_frequencies(128, 10000.0, YARN)
    inv, _ = decoder.rope_frequencies(128, 10000.0, dict(YARN, truncate=False))
    plain = 10000.0 ** (-2.0 * np.arange(64) / 128)
    ends = [128 * math.log(4096 / (2 * math.pi * t)) / (2 * math.log(10000.0)) for t in (32, 1)]
    ramp = np.clip((np.arange(64) - ends[0]) / (ends[1] - ends[0]), 0, 1)
    want = plain * (1 - ramp) + plain / 8 * ramp
    assert np.all(np.abs(inv - want) <= 2.0 ** -23 * want)
    assert not np.array_equal(whole, inv)
    same, _ = decoder.rope_frequencies(128, 10000.0, dict(YARN, truncate=True))
    assert np.array_equal(same, whole)


L3 = dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
          original_max_position_embeddings=8192)


@pytest.mark.parametrize("bad", [
    dict(L3, high_freq_factor=1.0), dict(L3, high_freq_factor=0.5), dict(L3, low_freq_factor=4.0),
    dict(L3, high_freq_factor=math.nan), dict(L3, original_max_position_embeddings=0),
    dict(L3, original_max_position_embeddings=-8192), dict(YARN, original_max_position_embeddings=0),
    dict(YARN, original_max_position_embeddings=math.nan), dict(YARN, beta_slow=0.0),
    dict(YARN, beta_fast=0.0), dict(YARN, beta_fast=1.0, beta_slow=32.0),
    dict(YARN, beta_fast=math.nan)])
def test_scalings_of_no_meaning_are_refused(bad):
    with pytest.raises(ValueError):
        decoder.rope_frequencies(64, 10000.0, bad)

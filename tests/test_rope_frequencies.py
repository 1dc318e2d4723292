"""Frequencies of rope_positions against the formulas, one pair at a time."""
import math

import numpy as np
import pytest

from ncmorph_amd import decoder

L3 = dict(rope_type="llama3", factor=32.0, low_freq_factor=1.0, high_freq_factor=4.0,
          original_max_position_embeddings=8192)
YARN = dict(type="yarn", factor=8.0, original_max_position_embeddings=4096)


def test_plain_linear_and_ntk():
    inv, scale = decoder.rope_frequencies(64, 10000.0)
    assert inv.dtype == np.float32 and scale == 1.0
    want = [10000.0 ** (-2 * p / 64) for p in range(32)]
    assert np.array_equal(inv, np.array(want, np.float32))
    lin, _ = decoder.rope_frequencies(64, 10000.0, dict(rope_type="linear", factor=4.0))
    assert np.array_equal(lin, np.array([w / 4.0 for w in want], np.float32))
    ntk, _ = decoder.rope_frequencies(64, 10000.0, dict(type="ntk", factor=4.0))
    assert ntk[0] == 1.0 and abs(ntk[-1] * 4.0 / inv[-1] - 1.0) < 1e-6


def test_llama3_is_the_decoders():
    """The decoder's own (every operation in float32): 8 roundings of 2^-24."""
    spec = decoder.DecoderSpec(hidden=64, intermediate=64, vocab=64, q_heads=1, kv_heads=1,
                               head_dim=64, layers=1)
    ref = decoder.rope_inverse_frequencies(spec).astype(np.float64)
    inv, scale = decoder.rope_frequencies(64, spec.rope_theta, L3)
    # powf of an exponent rounded to float32: ln(theta) 2^-25 more.
    assert np.all(np.abs(inv - ref) <= (8 + math.log(spec.rope_theta)) * 2.0 ** -24 * ref)
    assert scale == 1.0


def test_yarn():
    inv, scale = decoder.rope_frequencies(128, 10000.0, YARN)
    assert abs(scale - (0.1 * math.log(8.0) + 1.0)) < 1e-12
    plain, _ = decoder.rope_frequencies(128, 10000.0)
    turns = 4096 * plain / (2 * math.pi)
    ratio = inv / plain
    assert np.all(ratio[turns > 40] == 1.0)               # fast pairs as they are
    assert np.all(np.abs(ratio[turns < 0.8] - 0.125) < 1e-6)  # slow ones stretched
    assert np.all(np.diff(ratio) <= 1e-7)
    assert decoder.rope_frequencies(128, 1e4, dict(YARN, attention_factor=2.0))[1] == 2.0


@pytest.mark.parametrize("bad", [dict(type="dynamic", factor=2.0), dict(type="linear", factor=0.0),
                                 dict(type="linear", factor=float("nan"))])
def test_refused(bad):
    with pytest.raises(ValueError):
        decoder.rope_frequencies(64, 10000.0, bad)
    for rot, theta in ((0, 1e4), (7, 1e4), (64, 1.0), (64, float("nan"))):
        with pytest.raises(ValueError):
            decoder.rope_frequencies(rot, theta)

"""CPU: how far the 4-bit cache's offset is from the middle of its group's levels (tests/kv4_ref.py, the definition)."""
import numpy as np
import pytest

import kv4_ref as R


def read_back(x):
    codes, words = R.quantise(x)
    s, z = (R.of_bits(b).astype(np.float64) for b in (words >> 16, words & 0xFFFF))
    return (codes.astype(np.float64) - 8) * np.repeat(s, 64, -1) + np.repeat(z, 64, -1), s, z


def test_the_offset_rounds_by_up_to_2_to_the_minus_8():
    """bf16 has 8 significant bits: 1 + 2^-8 lies half way between 1 and 1 + 2^-7 and goes to the even one, 1."""
    back, _, z = read_back(np.full(64, 1 + 2.0 ** -8, np.float32))
    assert z[0] == 1 and np.all(np.abs(back - (1 + 2.0 ** -8)) <= 2.0 ** -8)
    assert np.all(np.abs(back - (1 + 2.0 ** -8)) > 2.0 ** -9 * (1 + 2.0 ** -8))


def test_constants_read_back_within_2_to_the_minus_8():
    x = np.exp2(np.random.default_rng(0).uniform(-40, 40, (5000, 1))).astype(np.float32).repeat(64, 1)
    back, _, _ = read_back(x)
    off = np.abs(back - x) / x
    assert off.max() <= 2.0 ** -8 and off.max() > 2.0 ** -9


@pytest.mark.parametrize("seed", [1, 2])
def test_codes_are_cut_off_only_far_from_zero(seed):
    """The levels reach half a step past lo and hi, and the offset's rounding is at most 2^-8 |z|: none is cut off where
    |z| is below 2^7 s (s is rounded up: hi may lie half a step and more inside)."""
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((20000, 64)) * np.exp2(rng.uniform(-10, 0, (20000, 1))) + 1).astype(np.float32)
    _, words = R.quantise(x)
    s, z = (R.of_bits(b).astype(np.float32) for b in (words >> 16, words & 0xFFFF))
    t = np.rint((x - z) * (np.float32(1) / s))
    cut = ((t < -8) | (t > 7)).any(-1)
    ratio = np.abs(z / s)[:, 0]
    assert cut.any() and not cut[ratio < 127].any()   # t's own two roundings: 2^-22 of 127

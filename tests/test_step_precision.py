"""The bounds of step_precision notice what they are for: the lesser step breaks each, in numpy."""
import numpy as np
import pytest

import step_precision as sp


def test_an_angle_rounded_to_32_bits_breaks_its_bound():
    at, f, c, s = sp.angle_cases()
    for got, want in zip(sp.angle_rounded(at, f), (c, s)):
        off = np.abs(got.astype(np.longdouble) - want).astype(np.float64)
        bound = sp.angle_bound(want.astype(np.float64), at, f)
        assert (off > bound).mean() > 0.02 and (off > 10 * bound).any()


@pytest.mark.parametrize("length", [11, 12, 13])
def test_a_logarithm_of_the_scores_size_breaks_the_weights_bound(length):
    off = [abs(sp.weight_by_logarithm(128 * x * np.log2(np.e), length) * length - 1) for x in sp.SIZES]
    assert max(off) > 5 * sp.weights_bound(1.0)


def test_equal_weights():
    assert np.allclose(sp.equal_weights(1, 16, 8), 0.5) and np.allclose(sp.equal_weights(3, 3, 2).sum(), 6)


@pytest.mark.parametrize("height", [20.0, 30.0])
def test_sums_in_32_bits_break_the_entropy_s_bound(height):
    x, at = sp.peaked(8, 20000, height)
    bound = sp.peaked_bound(x, at)
    for got, want in zip(sp.peaked_in_32_bits(x, at), sp.peaked_exact(x, at)):
        assert (np.abs(got - want) > 5 * bound * np.abs(want)).all()
    assert (bound < 4e-5).all()


def test_the_exact_entropy():
    x, at = sp.peaked(4, 500, 3.0)
    e = np.exp(x.astype(np.float64))
    p = e / e.sum(1, keepdims=True)
    h, lp = sp.peaked_exact(x, at)
    assert np.allclose(h, -(p * np.log(p)).sum(1)) and np.allclose(lp, np.log(p[np.arange(4), at]))

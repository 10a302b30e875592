"""norm_bounds against the oracle, and that its tolerances are tight enough to fail."""
import numpy as np
import pytest

pytest.importorskip('torch')

import norm_bounds  # noqa: E402
import operator_oracle as oracle  # noqa: E402


@pytest.mark.parametrize('activation', ['linear', 'sigmoid', 'tanh', 'silu'])
@pytest.mark.parametrize('groups,c,lengths,rate', [(3, 12, [9, 0, 4], 0.2), (5, 5, None, 0.0), (1, 8, [1, 9, 2], 0.5)])
def test_same_as_the_oracle(activation, groups, c, lengths, rate):
    rng = np.random.default_rng(4)
    x, grad, w, b = rng.normal(size=(3, 9, c)), rng.normal(size=(3, 9, c)), rng.normal(size=c), rng.normal(size=c)
    want = oracle.group_norm(x, groups, w, b, 1e-5, activation, lengths, rate, 77, 1 << 40, grad)
    norm = norm_bounds.Norm(x, groups, w, b, 1e-5, activation, lengths, rate, 77, 1 << 40)
    mean, rstd, _, _ = norm.statistics()
    y, bound = norm.forward(mean, rstd, 2.0 ** -24, 0.0)
    parts = norm.gradient(grad, mean, rstd, 2.0 ** -24, 0.0)
    for got, expected in zip((y, mean, rstd, *(p for p, _ in parts)), want):
        assert np.allclose(got, expected, rtol=1e-11, atol=1e-11)
    assert np.linalg.norm(bound) < 1e-4 * np.linalg.norm(y)
    for value, off in parts:
        assert np.linalg.norm(off) < 1e-3 * np.linalg.norm(value)


def test_level_far_above_the_spread_is_a_tight_test():
    """With the statistics given, a gradient without its mean terms is far outside the bounds."""
    rng = np.random.default_rng(5)
    x, grad = (1000 + rng.normal(size=(2, 3000, 16))).astype(np.float32).astype(np.float64), 1 + rng.normal(size=(2, 3000, 16))
    norm = norm_bounds.Norm(x, 2, None, None, 1e-5, 'linear', None, 0.0, 0, 0)
    mean, rstd, _, _ = norm.statistics()
    dx, bound = norm.gradient(grad, mean, rstd, 2.0 ** -24, 0.0)[0]
    assert np.linalg.norm(bound) < 0.01 * np.linalg.norm(dx)
    assert (abs(grad * rstd.mean() - dx) > bound).mean() > 0.9


def test_masks_by_whole_arrays():
    for count, rate, seed, offset in ((1, 0.5, 3, 4), (1001, 0.1, (1 << 63) + 5, (1 << 35) + 1), (64, 1.0, 0, 0)):
        got, want = norm_bounds.kept(count, rate, seed, offset), oracle.kept(count, rate, seed, offset)
        assert np.array_equal(got[0], want[0]) and got[1] == want[1]

"""The global norm and clipping of doubles whose squares are no doubles.  Tolerances: the norm of n values is a sum of n squares,
n 2^-53 at the very worst and four roundings; clipped values have three more."""
import numpy as np
import pytest

from cortex_b200 import optimize
from cortex_b200 import tensor as ct
from test_gpu_experts import stream  # noqa: F401

pytestmark = pytest.mark.gpu
U = 2.0 ** -53


def _norm(g):
    """In 64 bits, by the largest value."""
    m = np.abs(g).max(initial=0.0)
    return m * np.sqrt(np.sum((g / m) ** 2)) if m > 0 else 0.0


@pytest.mark.parametrize("n", [1, 3, 300, 4096, 70001])
@pytest.mark.parametrize("low,high", [(500, 1000), (-1000, -500), (-1020, -1010), (-700, 700), (470, 490), (-490, -470), (-5, 5)])
def test_norm_and_clipping_of_doubles_of_any_size(stream, n, low, high):  # noqa: F811
    rng = np.random.default_rng(n + low + 2000)
    g = rng.standard_normal(n) * np.exp2(rng.uniform(low, high, n))
    if n > 2:
        g[n // 2] = 0.0
    norm = _norm(g)
    t, c = ct.to_tensor(g, "double"), ct.new_tensor([n], "double")
    got = ct.to_array(optimize.global_norm([t]))[0]
    assert abs(got - norm) <= norm * (n + 4) * U
    # bounds far below the norm too: the scale itself may be below the normal range
    for bound in (norm * 0.25, min(norm * 4.0, 1e308), max(norm * 1e-290, 1e-300)):
        before = ct.to_array(optimize.clip_gradients([t], bound, clipped=[c]))[0]
        assert before == got
        want = g if norm <= bound else g / norm * bound
        # a result below the normal range is off by half its step, and so may what it is computed from have been
        assert np.all(np.abs(ct.to_array(c) - want) <= np.abs(want) * (n + 10) * U + 2.0 ** -1073 + np.abs(bound) * 2.0 ** -1074)


def test_doubles_without_a_finite_norm(stream):  # noqa: F811
    c = ct.new_tensor([3], "double")
    for bad in (np.inf, np.nan, -np.inf):
        for scale in (1.0, 1e200, 1e-200):
            data = np.array([scale, bad, 2 * scale])
            norm = ct.to_array(optimize.clip_gradients([ct.to_tensor(data, "double")], 1e-250, clipped=[c]))[0]
            assert not np.isfinite(norm) and np.array_equal(ct.to_array(c), data, equal_nan=True)
    huge = np.array([1.7e308, 1.7e308, 0.0])                 # finite values whose norm is no double: as the header says
    norm = ct.to_array(optimize.clip_gradients([ct.to_tensor(huge, "double")], 1.0, clipped=[c]))[0]
    assert np.isinf(norm) and np.array_equal(ct.to_array(c), huge)

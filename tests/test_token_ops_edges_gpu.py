"""The operators around an expert layer's products, and dropout: contents, sizes and uses at their edges, against plain 64-bit
forms.  Every input is made from fixed numbers.  Tolerances as in test_token_ops_gpu.py."""
import numpy as np
import pytest

import test_token_ops_gpu as base
import token_ref as R
from token_ref import EPS, device_matrix, host, out_slack

pytestmark = pytest.mark.gpu

LARGEST = {"f32": 3.4028234663852886e38, "bf16": 3.3895313892515355e38, "f16": 65504.0}


def rng(*key):
    return np.random.Generator(np.random.PCG64([int(k) for k in key]))


# ------------------------------------------------------------------------------------------------ router


@pytest.mark.parametrize("scoring,normalize", base.MODES)
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_infinite_logits_count_as_the_largest_value_forward_and_backward(gpu, dtype, scoring, normalize):
    """+inf is chosen before the largest finite value and weighs as much, in the weights and in their gradient"""
    inf, big = np.inf, LARGEST[dtype]
    near = 65472.0 if dtype == "f16" else 1.0  # 32 below the largest: an exponential that is not zero
    rows = np.array([[inf, big, 1, -inf, 0], [big, inf, 2, big, near], [inf, inf, -big, np.nan, near], [inf, 0, 1, 2, -1],
                     [-big, -inf, inf, -big, 3], [inf] * 5])
    logits = device_matrix(rows, dtype)
    x = host(logits)
    assert np.array_equal(np.isinf(x), np.isinf(rows))  # the values are the type's own
    finite = np.where(x == inf, big, x)
    w, idx = base.run_route(gpu[0], logits, 3, scoring, normalize)
    assert np.array_equal(idx, R.choose(x, 3))
    want = R.route_weights(finite, idx, scoring, normalize, 1.0)
    # arguments of exponentials are 0, -32 or beyond any share
    base.check(w, want, np.abs(want) * EPS * (2 * (2 + 32) + 32 + 5 + 6) + 2.0 ** -126)
    g = rng(31).standard_normal((len(rows), 3)).astype(np.float32).astype(np.float64)
    with np.errstate(over="ignore"):
        want, size = R.route_backward(finite, idx, g, scoring, normalize, 1.5)
    got = base.run_route_backward(gpu[0], logits, idx, g, scoring, normalize, 1.5)
    base.check(got, want, size * EPS * (4 * (2 + 32) + 64 + 3) + out_slack(want, dtype) + 2.0 ** -126)


@pytest.mark.parametrize("scoring,normalize", base.MODES)
def test_f16_masks_ties_and_lowest_values(gpu, scoring, normalize):
    """16-bit values of that format have keys of their own: signed zeros, ties, masks, the lowest value"""
    inf, nan, low = np.inf, np.nan, -65504.0
    rows = np.array([[-inf] * 6, [1, -inf, -inf, -inf, -inf, -inf], [nan, 2, nan, 1, -inf, -inf], [nan] * 6, [0.0, -0.0, 0.0, -0.0, 0.0, -0.0],
                     [1, 1, 1, 1, 1, 1], [low] * 6, [low, 1, low, low, 2, low], [-200, -200, -300, -250, -400, -1000],
                     [3, 1, 3, 1, 3, 1], [88, -88, 0, 100, -100, 50], [6e-8, -6e-8, 0, -0.0, 6e-5, -6e-5]])
    logits = device_matrix(rows, "f16")
    x = host(logits)
    w, idx = base.run_route(gpu[0], logits, 4, scoring, normalize)
    assert np.array_equal(idx, R.choose(x, 4))
    want = R.route_weights(x, idx, scoring, normalize, 1.0)
    usual = np.array([np.abs(v[np.isfinite(v)]).max(initial=0) < 2000 for v in x])
    base.check(w[usual], want[usual], base.weight_bound(x[usual], want[usual]))
    base.check(w[~usual], want[~usual], np.abs(want[~usual]) * 64 * EPS + 2.0 ** -126)
    d = base.run_route_backward(gpu[0], logits, idx, np.ones((len(rows), 4)), scoring, normalize)
    assert np.isfinite(d).all() and not d[np.isnan(x) | (x == -inf)].any()

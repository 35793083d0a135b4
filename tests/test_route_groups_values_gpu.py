"""The router with groups of experts on a device where scores are at the lower end of 32 bits."""
import numpy as np
import pytest

import layer_ref as L
import token_ref as R
from test_route_groups_gpu import run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bias", [None, 0.0])
def test_groups_of_the_smallest_scores(gpu, bias):
    """sums of scores near the least normal number and below it: sigmoids of logits of -87, a softmax's scores 100 below the best"""
    sigmoid = [[-87, -100, -87.4, -87.4], [-87.25, -87.4, -87.2, -90], [-88, -88, -87.8, -89], [-95, -95, -94.5, -97], [-103, -103, -102.6, -120],
               [-120, -120, -119.5, -140]]
    softmax = [[0, -50, -103.5, -103.5, -102.9, -104], [0, -50, -100, -100, -99.5, -102], [0, -1, -92, -95, -92.5, -92.5],
               [0, 0, -104, -104, -103.5, -106], [0, -3, -130, -130, -129.5, -140]]
    for scoring, rows, groups, kept in (("sigmoid", sigmoid, 2, 1), ("softmax", softmax, 3, 2)):
        x = np.array(rows).astype(np.float32).astype(np.float64)
        b = None if bias is None else np.full(x.shape[1], bias)
        for best in (1, 2):
            for order in (slice(None), slice(None, None, -1)):  # the better group first and last
                logits = np.ascontiguousarray(x[:, order])
                _, idx = run(gpu, R.device_matrix(logits, "f32"), b, 2 * kept, scoring, True, 1.0, groups, kept, best)
                assert np.array_equal(idx, L.choose(logits, b, scoring, 2 * kept, groups, kept, best)), (scoring, best)


@pytest.mark.parametrize("scoring,dtype", [("softmax", "f32"), ("softmax", "bf16"), ("sigmoid", "f32"), ("sigmoid", "bf16")])
@pytest.mark.parametrize("E,groups,kept,best", [(32, 8, 3, 2), (60, 5, 2, 2), (64, 8, 4, 1), (40, 1, 1, 1)])
def test_many_rows_of_the_smallest_scores(gpu, scoring, dtype, E, groups, kept, best):
    """as many groups as are kept less one have an expert of an ordinary score; the others are of scores down to nothing"""
    r = np.random.Generator(np.random.PCG64([E, groups]))
    T = 800
    x = -r.uniform(84, 112, (T, 1)) + r.standard_normal((T, E)) * r.choice([0.25, 1.0, 4.0], (T, 1))
    for g in range(kept - 1):
        x[:, g * (E // groups)] = r.standard_normal(T)
    if scoring == "softmax":
        x[:, 0] = 0
    logits = R.device_matrix(x, dtype)
    _, idx = run(gpu, logits, np.zeros(E) if groups == 1 else None, 4, scoring, True, 1.0, groups, kept, best)
    want = L.choose(R.host(logits), None, scoring, 4, groups, kept, best)
    bad = (idx != want).any(1)
    assert not bad.any(), (bad.sum(), np.argwhere(bad)[:5], idx[bad][:3], want[bad][:3])


@pytest.mark.parametrize("scoring,dtype", [("softmax", "f32"), ("sigmoid", "f16"), ("sigmoid", "bf16")])
@pytest.mark.parametrize("E,groups,kept", [(16, 8, 3), (20, 5, 3), (24, 8, 6), (32, 16, 11), (256, 8, 4)])
@pytest.mark.parametrize("lowest", [-np.finfo(np.float32).max, -1e38, -1e30])
def test_biases_that_mask_by_a_low_value(gpu, scoring, dtype, E, groups, kept, lowest):
    """Groups whose best two have such a bias come behind all others, and in front of those in which every expert is masked: their
    sum of two is beyond 32 bits."""
    r = np.random.Generator(np.random.PCG64([E, groups]))
    T, size = 300, E // groups
    x = r.standard_normal((T, E))
    x[(r.random((T, groups)) < 0.4).repeat(size, 1)] = -np.inf
    x[r.random((T, E)) < 0.2] = np.nan
    logits = R.device_matrix(x, dtype)
    for share in (0.3, 0.9, 1.0):
        bias = (0.1 * r.standard_normal(E)).astype(np.float32).astype(np.float64)
        bias[(r.random(groups) < share).repeat(size)] = float(np.float32(lowest))
        for best in (1, 2):
            _, idx = run(gpu, logits, bias, kept * size if E <= 32 else 8, scoring, True, 1.0, groups, kept, best)
            want = L.choose(R.host(logits), bias, scoring, kept * size if E <= 32 else 8, groups, kept, best)
            bad = (idx != want).any(1)
            assert not bad.any(), (share, best, bad.sum(), np.argwhere(bad)[:3].ravel(), idx[bad][:2], want[bad][:2])

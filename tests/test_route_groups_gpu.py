"""The router with a bias on the choice and groups of experts on a device, against the 64-bit form (layer_ref.py)."""
import numpy as np
import pytest

import layer_ref as L
import token_ref as R
from test_token_ops_gpu import check, run_route_backward, weight_bound

pytestmark = pytest.mark.gpu

MODES = [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)]


def run(gpu, logits, bias, k, scoring, normalize=True, scale=1.0, groups=1, kept=1, best=1, c=None):
    import torch
    from onednn_b200 import api
    c = c or R.Call(gpu[0])
    T = logits.shape[0]
    w = torch.full((T, k), 7.0, device="cuda:0")
    i = torch.full((T, k), 7, dtype=torch.int32, device="cuda:0")
    b = None if bias is None else c.bind(api.ARG_BIAS, R.device_matrix(bias[None, :], "f32")[0])
    pd = api.moe_route.primitive_desc(
        gpu[0], c.bind(api.ARG_SRC, logits), c.bind(api.ARG_DST, w), c.bind(api.ARG_DST_1, i), scoring=getattr(api.scoring, scoring),
        normalize=normalize, scale=scale, bias_md=b, groups=groups, groups_kept=kept, group_best=best)
    c.run(api.moe_route, pd).strm.wait()
    return R.host(w), R.host(i)


def case(*seed):
    return np.random.Generator(np.random.PCG64([sum(map(ord, str(s))) for s in seed]))


# (T, E, k, groups, kept, best): every number of values a lane can hold, groups of one and of all, sizes that are no power of two
SHAPES = [(1, 256, 8, 8, 4, 2), (70, 256, 8, 8, 4, 2), (33, 160, 6, 8, 3, 1), (9, 64, 4, 1, 1, 1), (40, 60, 5, 6, 2, 2), (7, 12, 12, 3, 3, 1),
          (21, 512, 8, 16, 4, 2), (13, 1024, 32, 32, 8, 2), (19, 33, 3, 33 // 11, 1, 2), (5, 32, 2, 32, 2, 2), (11, 1, 1, 1, 1, 2),
          (6, 1000, 7, 5, 2, 1), (17, 130, 4, 2, 1, 2)]


@pytest.mark.parametrize("scoring,normalize", MODES)
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("T,E,k,groups,kept,best", SHAPES)
def test_route(gpu, T, E, k, groups, kept, best, dtype, scoring, normalize):
    r = case(T, E, k, dtype)
    logits = R.device_matrix(r.standard_normal((T, E)) * 2, dtype, pitch=E + T % 3, offset=T % 2)
    bias = (r.standard_normal(E) * (0.1 if scoring == "sigmoid" else 0.3 / E)).astype(np.float32).astype(np.float64)
    x = R.host(logits)
    for b in (bias, None):
        w, idx = run(gpu, logits, b, k, scoring, normalize, 2.5, groups, kept, best)
        want_idx = L.choose(x, b, scoring, k, groups, kept, best)
        assert np.array_equal(idx, want_idx)
        want = R.route_weights(x, want_idx, scoring, normalize, 2.5)
        check(w, want, weight_bound(x, want))


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_masks_ties_and_infinities(gpu, dtype, scoring):
    inf, nan = np.inf, np.nan
    rows = [[-inf] * 8, [1, -inf, -inf, -inf, -inf, -inf, -inf, -inf], [nan, 2, nan, 1, -inf, -inf, 0, nan], [nan] * 8,
            [0.0, -0.0] * 4, [1] * 8, [-200, -200, -300, -250, -400, -1000, -500, -500], [3, 1, 3, 1, 3, 1, 3, 1],
            [40, 50, 60, 70, 80, 90, 100, 110], [-inf, -inf, 5, 4, 5, 4, -inf, -inf], [20, 21, 22, 23, 24, 25, 26, 27]]
    logits = R.device_matrix(np.array(rows), dtype)
    x = R.host(logits)
    for b in (None, [0.0] * 8, [0, 0, 0.5, 0.5, 0, 0, 0.25, 0.25], [-inf, 0, nan, 0, 0, 0, 0, 0], [-3, -2, -1, -1, -2, -3, -0.5, -0.5],
              [inf, 0, 0, inf, 0, 0, 0, 0], [nan] * 8, [-inf, -inf, 0, 0, 0, 0, -inf, -inf]):
        b = None if b is None else np.array(b, float)
        for groups, kept, best in ((1, 1, 1), (4, 2, 2), (4, 2, 1), (2, 1, 2), (8, 4, 2)):
            w, idx = run(gpu, logits, b, 4, scoring, True, 1.0, groups, kept, best)
            want_idx = L.choose(x, None if b is None else np.where(np.isnan(b), -inf, b), scoring, 4, groups, kept, best)
            if b is None and groups == 1:  # the plain router: by the logits, which differ where sigmoids are all 1
                want_idx = R.choose(x, 4)
            assert np.array_equal(idx, want_idx), (b, groups, kept, best, idx, want_idx)
            want = R.route_weights(x, want_idx, scoring, True, 1.0)
            usual = np.abs(np.where(np.isfinite(x), x, 0)).max(1) < 600
            check(w[usual], want[usual], weight_bound(x[usual], want[usual]))


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,groups,kept", [(64, 1, 1), (256, 8, 4), (160, 8, 3)])
def test_choices_that_32_bits_do_not_tell(gpu, E, groups, kept, scoring):
    """values around the choice differ by some 2^-30: scores of neighbouring logits and biases that undo the difference"""
    r = case(E, groups, scoring)
    T = 64
    x = (r.standard_normal((T, 1)) * 0.5 + np.arange(E)[None, :] * 2.0 ** -22 * r.choice([-1, 1], (1, E))).astype(np.float32).astype(np.float64)
    logits = R.device_matrix(x, "f32")
    bias = (r.integers(-8, 9, E) * 2.0 ** -27).astype(np.float32).astype(np.float64)
    for b in (bias, None):
        _, idx = run(gpu, logits, b, 6, scoring, True, 1.0, groups, kept, 2)
        assert np.array_equal(idx, L.choose(x, b, scoring, 6, groups, kept, 2))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_many_rows(gpu, dtype):
    """a full batch: what 32 bits decide and what they leave open, side by side"""
    r = case(dtype)
    T, E = 6000, 256
    logits = R.device_matrix(r.standard_normal((T, E)), dtype)
    bias = (0.05 * r.standard_normal(E)).astype(np.float32).astype(np.float64)
    x = R.host(logits)
    for scoring in ("sigmoid", "softmax"):
        b = bias if scoring == "sigmoid" else (bias / 100).astype(np.float32).astype(np.float64)
        _, idx = run(gpu, logits, b, 8, scoring, True, 1.0, 8, 4, 2)
        assert np.array_equal(idx, L.choose(x, b, scoring, 8, 8, 4, 2))


@pytest.mark.parametrize("scoring,normalize", MODES)
def test_the_gradient_takes_the_indices(gpu, scoring, normalize):
    r = case(5)
    T, E, k = 20, 64, 6
    logits = R.device_matrix(r.standard_normal((T, E)), "f32")
    x = R.host(logits)
    bias = (0.3 * r.standard_normal(E)).astype(np.float32).astype(np.float64)
    _, idx = run(gpu, logits, bias, k, scoring, normalize, 2.5, 8, 3, 2)
    g = r.standard_normal((T, k)).astype(np.float32).astype(np.float64)
    want, size = R.route_backward(x, idx, g, scoring, normalize, 2.5)
    got = run_route_backward(gpu[0], logits, idx, g, scoring, normalize, 2.5)
    check(got, want, size * L.EPS * (4 * (2 + x.max() - x.min()) + 64 + k) + 2.0 ** -140)


def test_open_dims_and_a_captured_graph(gpu):
    import torch
    from onednn_b200 import api
    E, k = 48, 4
    r = case(6)
    bias = (0.1 * r.standard_normal(E)).astype(np.float32).astype(np.float64)
    prim = None
    for T in (3, 100, 0):
        x = r.standard_normal((T, E)).astype(np.float32).astype(np.float64)
        c = R.Call(gpu[0])
        w, i = torch.empty((T, k), device="cuda:0"), torch.empty((T, k), dtype=torch.int32, device="cuda:0")
        mds = [c.bind(a, t, (0,)) for a, t in ((api.ARG_SRC, R.device_matrix(x, "f32")), (api.ARG_DST, w), (api.ARG_DST_1, i))]
        bmd = c.bind(api.ARG_BIAS, R.device_matrix(bias[None], "f32")[0])
        prim = prim or api.moe_route(api.moe_route.primitive_desc(gpu[0], *mds, bias_md=bmd, groups=6, groups_kept=2, group_best=2,
                                                                  scoring=api.scoring.sigmoid))
        prim.execute(c.strm, c.args)
        c.strm.wait()
        assert np.array_equal(R.host(i), L.choose(x, bias, "sigmoid", k, 6, 2, 2))
    s = torch.cuda.Stream()
    c = R.Call(gpu[0], s.cuda_stream)
    logits = torch.empty((30, E), device="cuda:0")
    w, i = torch.empty((30, k), device="cuda:0"), torch.empty((30, k), dtype=torch.int32, device="cuda:0")
    for arg, t in ((api.ARG_SRC, logits), (api.ARG_DST, w), (api.ARG_DST_1, i), (api.ARG_BIAS, R.device_matrix(bias[None], "f32")[0])):
        c.bind(arg, t)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        prim.execute(c.strm, c.args)
    for _ in range(2):
        x = r.standard_normal((30, E)).astype(np.float32)
        logits.copy_(torch.from_numpy(x))
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(R.host(i), L.choose(x.astype(np.float64), bias, "sigmoid", k, 6, 2, 2))

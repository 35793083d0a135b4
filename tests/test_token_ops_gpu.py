"""The operators around an expert layer's products, and dropout, on the device against plain 64-bit forms.

Tolerances: integers and copies are equal.  With u = 2^-24: an exponential is within 2 units and carries its argument's
rounding (|argument| u); a sum of n terms is within n u of the sum of magnitudes; each product or quotient adds u; a result
stored in fewer bits adds half a unit of its type."""
import numpy as np
import pytest

import token_ref as R
from token_ref import EPS, Call, device_matrix, host, out_slack

pytestmark = pytest.mark.gpu


def rng(*key):
    return np.random.Generator(np.random.PCG64([abs(hash(k)) % (1 << 31) if isinstance(k, str) else int(k) for k in key]))


def check(got, want, bound):
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), "%d of %d beyond the bound, first at %s: %s for %s within %s" % (
        bad.sum(), bad.size, np.argwhere(bad)[0], got[bad][0], want[bad][0], bound[bad][0])


# ------------------------------------------------------------------------------------------------ router

SHAPES = [(1, 1, 1), (1, 64, 8), (3, 7, 7), (5, 33, 4), (130, 100, 6), (67, 256, 8), (9, 1000, 32), (4, 1024, 1),
          (515, 160, 6), (2, 512, 32)]
MODES = [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)]


def run_route(eng, logits, k, scoring, normalize, scale=1.0):
    import torch
    c = Call(eng)
    w = torch.full((logits.shape[0], k), 7.0, device="cuda:0")
    i = torch.full((logits.shape[0], k), 7, device="cuda:0", dtype=torch.int32)
    a = c.api
    pd = a.moe_route.primitive_desc(eng, c.bind(a.ARG_SRC, logits), c.bind(a.ARG_DST, w), c.bind(a.ARG_DST_1, i),
                                    scoring=getattr(a.scoring, scoring), normalize=normalize, scale=scale)
    c.run(a.moe_route, pd).strm.wait()
    return host(w), host(i)


def run_route_backward(eng, logits, idx, g, scoring, normalize, scale=1.0):
    import torch
    c = Call(eng)
    a = c.api
    d = torch.full_like(logits, 7.0)
    pd = a.moe_route_backward.primitive_desc(
        eng, c.bind(a.ARG_SRC, logits), c.bind(a.ARG_SRC_1, torch.from_numpy(idx).cuda()),
        c.bind(a.ARG_DIFF_DST, torch.from_numpy(g.astype(np.float32)).cuda()), c.bind(a.ARG_DIFF_SRC, d),
        scoring=getattr(a.scoring, scoring), normalize=normalize, scale=scale)
    c.run(a.moe_route_backward, pd).strm.wait()
    return host(d)


def weight_bound(logits, want, extra=0):
    """an exponential (twice: of the value and, summed, of the others), a sum over a lane's share and the lanes, a quotient
    and a product; the argument of an exponential is a difference of two logits"""
    finite = logits[np.isfinite(logits)]
    spread = (finite.max() - finite.min()) if finite.size else 0.0
    return np.abs(want) * EPS * (2 * (2 + spread) + 32 + 5 + 6 + extra) + 2.0 ** -140


@pytest.mark.parametrize("scoring,normalize", MODES)
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("T,E,k", SHAPES)
def test_route(gpu, T, E, k, dtype, scoring, normalize):
    r = rng(T, E, k, dtype)
    logits = device_matrix(r.standard_normal((T, E)) * 2, dtype, pitch=E + T % 3, offset=T % 2)
    x = host(logits)
    w, idx = run_route(gpu[0], logits, k, scoring, normalize, 2.5)
    want_idx = R.choose(x, k)
    assert np.array_equal(idx, want_idx)
    want = R.route_weights(x, want_idx, scoring, normalize, 2.5)
    check(w, want, weight_bound(x, want))


@pytest.mark.parametrize("scoring,normalize", MODES)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_route_masks_ties_and_infinities(gpu, dtype, scoring, normalize):
    inf, nan = np.inf, np.nan
    low = {"f32": -3.4028234663852886e38, "bf16": -3.3895313892515355e38}[dtype]
    rows = [[-inf] * 6, [1, -inf, -inf, -inf, -inf, -inf], [nan, 2, nan, 1, -inf, -inf], [nan] * 6, [0.0, -0.0, 0.0, -0.0, 0.0, -0.0],
            [1, 1, 1, 1, 1, 1], [low] * 6, [low, 1, low, low, 2, low], [-200, -200, -300, -250, -400, -1000],
            [3, 1, 3, 1, 3, 1], [88, -88, 0, 100, -100, 50]]
    logits = device_matrix(np.array(rows), dtype)
    x = host(logits)
    w, idx = run_route(gpu[0], logits, 4, scoring, normalize)
    want_idx = R.choose(x, 4)
    assert np.array_equal(idx, want_idx)
    want = R.route_weights(x, want_idx, scoring, normalize, 1.0)
    # the lowest row of the type spreads the arguments beyond any bound; its weights are 0, 1 or equal shares
    usual = np.array([np.abs(v[np.isfinite(v)]).max(initial=0) < 2000 for v in x])
    check(w[usual], want[usual], weight_bound(x[usual], want[usual]))
    check(w[~usual], want[~usual], np.abs(want[~usual]) * 64 * EPS + 2.0 ** -126)
    d = run_route_backward(gpu[0], logits, idx, np.ones((len(rows), 4)), scoring, normalize)
    assert np.isfinite(d).all() and not d[np.isnan(x) | (x == -inf)].any()


def test_route_infinite_logit(gpu):
    logits = device_matrix(np.array([[1.0, np.inf, 0.0, -np.inf]]), "f32")
    w, idx = run_route(gpu[0], logits, 4, "softmax", True)
    assert idx.tolist() == [[1, 0, 2, -1]] and w.tolist() == [[1.0, 0.0, 0.0, 0.0]]


@pytest.mark.parametrize("scoring,normalize", MODES)
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("T,E,k", SHAPES)
def test_route_backward(gpu, T, E, k, dtype, scoring, normalize):
    r = rng(T, E, k, dtype, 1)
    logits = device_matrix(r.standard_normal((T, E)), dtype, pitch=E + 1)
    x = host(logits)
    idx = R.choose(x, k)
    if T > 2:
        idx[1, k // 2:] = -1  # choices a program took back
    g = r.standard_normal((T, k)).astype(np.float32).astype(np.float64)
    want, size = R.route_backward(x, idx, g, scoring, normalize, 2.5)
    got = run_route_backward(gpu[0], logits, idx, g, scoring, normalize, 2.5)
    spread = x.max() - x.min()
    check(got, want, size * EPS * (4 * (2 + spread) + 64 + k) + out_slack(want, dtype) + 2.0 ** -140)


@pytest.mark.parametrize("scoring,normalize", MODES)
def test_route_backward_against_differences(gpu, scoring, normalize):
    """<gradient, v> equals the central difference of the 64-bit forward along v (step h: error of order h^2)"""
    r = rng(11)
    T, E, k, h = 6, 40, 5, 1e-5
    logits = device_matrix(r.standard_normal((T, E)), "f32")
    x, g, v = host(logits), r.standard_normal((T, k)).astype(np.float32).astype(np.float64), r.standard_normal((T, E))
    idx = R.choose(x, k)
    d = run_route_backward(gpu[0], logits, idx, g, scoring, normalize, 1.5)
    f = [(R.route_weights(x + s * h * v, idx, scoring, normalize, 1.5) * g).sum() for s in (1, -1)]
    _, size = R.route_backward(x, idx, g, scoring, normalize, 1.5)
    # (third derivatives of these functions are below 10 per direction component)
    bound = (size * np.abs(v)).sum() * EPS * 128 + 10 * h * h * np.abs(g).sum() * np.abs(v).max() ** 3 * E
    assert abs((d * v).sum() - (f[0] - f[1]) / (2 * h)) <= bound


# ---------------------------------------------------------------------------------------------- dispatch


def choices(r, T, E, k, dropped):
    idx = np.argsort(r.random((T, E)) * (0.2 + r.random(E)), axis=1)[:, :k].astype(np.int32) if T * E < 5e6 else \
        r.integers(0, E, (T, k)).astype(np.int32)
    if dropped:
        out = r.random((T, k)) < dropped
        idx[out] = r.choice(np.array([-1, E, -2 ** 31, 2 ** 31 - 1, E + 7]), out.sum())
    return idx


def run_dispatch(eng, x, idx, E, idx_pitch=0):
    import torch
    c = Call(eng)
    a = c.api
    T, H = x.shape
    k = idx.shape[1]
    rows = torch.full((T * k, H), 7, device="cuda:0", dtype=x.dtype)
    offsets = torch.full((E,), 7, device="cuda:0", dtype=torch.int32)
    pos = torch.full((T, k), 7, device="cuda:0", dtype=torch.int32)
    di = device_matrix(idx, "s32", idx_pitch)
    pd = a.moe_dispatch.primitive_desc(eng, c.bind(a.ARG_SRC, x), c.bind(a.ARG_SRC_1, di), c.grouped(a.ARG_DST, rows, offsets),
                                       c.bind(a.ARG_DST_1, pos))
    c.run(a.moe_dispatch, pd).strm.wait()
    return rows, offsets, pos


@pytest.mark.parametrize("T,E,k,H,dtype,dropped,pitch", [
    (1, 8, 2, 64, "bf16", 0, 0), (1, 1, 1, 1, "f32", 0, 0), (37, 8, 2, 4096, "bf16", 0, 0), (37, 8, 2, 4096, "bf16", 0.3, 4104),
    (300, 64, 8, 100, "f16", 0.1, 0), (256, 64, 8, 48, "bf16", 0, 0), (257, 64, 8, 48, "bf16", 0, 0), (5000, 5, 1, 7, "s8", 0.05, 0),
    (700, 160, 6, 2047, "f16", 0.15, 2053), (1025, 1024, 2, 33, "f32", 0, 0), (3000, 700, 4, 96, "s8", 0.5, 0),
    (20000, 64, 8, 16, "bf16", 0.01, 0), (9001, 1000, 32, 3, "f32", 0.2, 5), (2048, 1, 1, 8, "bf16", 0, 0), (64, 4, 2, 128, "f32", 1.0, 0),
    (2500, 3, 2, 130, "bf16", 1.0, 0)])
def test_dispatch(gpu, T, E, k, H, dtype, dropped, pitch):
    r = rng(T, E, k, H)
    k = min(k, E)
    x = device_matrix(r.integers(-100, 100, (T, H)).astype(np.float64), dtype, pitch, offset=1 if pitch % 2 else 0)
    idx = choices(r, T, E, k, dropped)
    rows, offsets, pos = run_dispatch(gpu[0], x, idx, E, k + T % 3)
    ends, want_pos, order = R.sort_slots(idx, E)
    assert np.array_equal(host(offsets), ends)
    assert np.array_equal(host(pos), want_pos)
    want = np.zeros((T * k, H))
    want[:order.size] = host(x)[order // k]
    assert np.array_equal(host(rows), want)


def test_dispatch_all_to_one_expert_and_repeated_choices(gpu):
    r = rng(5)
    x = device_matrix(r.integers(-100, 100, (900, 24)).astype(np.float64), "bf16")
    idx = np.full((900, 4), 17, np.int32)
    rows, offsets, pos = run_dispatch(gpu[0], x, idx, 40)
    assert host(offsets).tolist() == [0] * 17 + [3600] * 23
    assert np.array_equal(host(pos).reshape(-1), np.arange(3600))
    assert np.array_equal(host(rows), np.repeat(host(x), 4, 0))


@pytest.mark.parametrize("T,H", [(0, 64), (5, 0), (3000, 0)])
def test_dispatch_of_nothing(gpu, T, H):
    import torch
    r = rng(T, H)
    idx = choices(r, T, 9, 2, 0.2)
    rows, offsets, pos = run_dispatch(gpu[0], torch.zeros((T, H), device="cuda:0"), idx, 9)
    ends, want_pos, _ = R.sort_slots(idx, 9)
    assert np.array_equal(host(offsets), ends) and np.array_equal(host(pos), want_pos)


# ----------------------------------------------------------------------------------------------- combine


def make_rows(r, T, E, k, H, dtype, dropped):
    import torch
    idx = choices(r, T, E, min(k, E), dropped) if k <= E else r.integers(0, E, (T, k)).astype(np.int32)
    ends, pos, _ = R.sort_slots(idx, E)
    rows = device_matrix(r.standard_normal((T * k, H)), dtype)
    return rows, torch.from_numpy(ends).cuda(), torch.from_numpy(pos).cuda(), pos


def run_combine(eng, rows, offsets, pos, out_dtype, weights=None, residual=None, p=0.0, seed=None, pitch=0):
    import torch
    c = Call(eng)
    a = c.api
    T = pos.shape[0]
    y = device_matrix(np.full((T, rows.shape[1]), 7.0), out_dtype, pitch)
    if seed is not None:
        c.bind(a.ARG_ATTR_DROPOUT_SEED, torch.tensor(seed, dtype=torch.int64, device="cuda:0"))
    pd = a.moe_combine.primitive_desc(eng, c.grouped(a.ARG_SRC, rows, offsets), c.bind(a.ARG_SRC_1, pos), c.bind(a.ARG_DST, y),
                                      weights_md=c.bind(a.ARG_WEIGHTS, weights), residual_md=c.bind(a.ARG_SRC_2, residual), dropout_p=p)
    c.run(a.moe_combine, pd).strm.wait()
    return host(y)


def combine_want(rows, pos, weights, residual, p, seed):
    x = host(rows)
    picked = np.where(pos[:, :, None] >= 0, x[np.maximum(pos, 0)], 0.0)
    w = weights[:, :, None] if weights is not None else 1.0
    terms = w * picked
    y, size = terms.sum(1), np.abs(terms).sum(1)
    if p:
        y, size = R.dropout(y, p, *seed), R.dropout(size, p, *seed)
    if residual is not None:
        y, size = y + residual, size + np.abs(residual)
    return y, size


COMBINE = [
    (1, 64, 8, 4096, "bf16", "bf16", True, True, 0.0, 0, 0), (1, 4, 1, 1, "f32", "f32", False, False, 0.0, 0, 0),
    (37, 8, 2, 100, "bf16", "f32", True, False, 0.3, 0, 0.2), (37, 8, 2, 104, "bf16", "bf16", True, True, 0.3, 120, 0.2),
    (19, 16, 9, 127, "f16", "f16", True, True, 0.5, 0, 0.1), (300, 64, 8, 2047, "f16", "f16", True, True, 0.1, 2053, 0.3),
    (33, 40, 32, 64, "f32", "bf16", True, True, 0.0, 0, 0), (64, 3, 3, 7, "f32", "f32", False, True, 0.25, 0, 0.5),
    (130, 8, 2, 1024, "bf16", "f16", False, False, 0.0, 0, 0.1), (11, 8, 4, 512, "f32", "f16", True, True, 1.0, 0, 0),
    (5, 8, 2, 2050, "bf16", "bf16", True, True, 0.2, 0, 1.0), (777, 32, 6, 8, "f16", "bf16", True, True, 0.1, 0, 0),
    (3, 4, 2, 1001, "f16", "f32", True, True, 0.4, 0, 0),
    # many tokens of wide rows: the form that streams them through shared memory (several tokens an item, several
    # segments a token, few and many stages, ragged last items and segments)
    (2050, 16, 8, 1024, "bf16", "bf16", True, True, 0.2, 0, 0.1), (2101, 16, 3, 1032, "f16", "f32", True, True, 0.0, 1040, 0.3),
    (700, 40, 32, 3080, "f32", "f16", True, True, 0.1, 0, 0), (1000, 8, 1, 2600, "bf16", "f16", False, False, 0.3, 0, 0),
    (601, 16, 8, 4104, "bf16", "bf16", True, True, 0.0, 0, 1.0), (530, 8, 5, 4352, "f32", "f32", True, False, 0.5, 0, 0.2),
    (1201, 32, 17, 1800, "bf16", "bf16", True, True, 0.0, 0, 0.05)]


@pytest.mark.parametrize("T,E,k,H,dtype,out,weighted,res,p,pitch,dropped", COMBINE)
def test_combine(gpu, T, E, k, H, dtype, out, weighted, res, p, pitch, dropped):
    import torch
    r = rng(T, E, k, H)
    rows, offsets, dpos, pos = make_rows(r, T, E, k, H, dtype, dropped)
    rows[int(offsets[-1]):] = float("nan")  # belong to no slot: never read
    weights = r.random((T, k)).astype(np.float32) if weighted else None
    if weighted and (pos < 0).any():
        weights[pos < 0] = np.inf  # of a slot without a row: not used
    residual = device_matrix(r.standard_normal((T, H)), out, pitch) if res else None
    seed = (int(r.integers(0, 2 ** 62)), int(r.integers(0, 2 ** 62))) if p else None
    got = run_combine(gpu[0], rows, offsets, dpos, out, torch.from_numpy(weights).cuda() if weighted else None, residual, p, seed, pitch)
    w = np.where(pos >= 0, weights, 0.0).astype(np.float64) if weighted else None
    want, size = combine_want(rows.nan_to_num(0.0), pos, w, host(residual) if res else None, p, seed)
    check(got, want, size * EPS * (k + 4) + out_slack(want, out))


@pytest.mark.parametrize("T,E,k,H,dtype,out,weighted,res,p,pitch,dropped", COMBINE)
def test_combine_backward(gpu, T, E, k, H, dtype, out, weighted, res, p, pitch, dropped):
    import torch
    r = rng(T, E, k, H, 3)
    rows, offsets, dpos, pos = make_rows(r, T, E, k, H, dtype, dropped)
    weights = r.standard_normal((T, k)).astype(np.float32)
    dy = device_matrix(r.standard_normal((T, H)), out, pitch)
    c = Call(gpu[0])
    a = c.api
    drows, dw = torch.full_like(rows, 7.0), torch.full((T, k), 7.0, device="cuda:0")
    seed = (int(r.integers(0, 2 ** 62)), int(r.integers(0, 2 ** 62)))
    if p:
        c.bind(a.ARG_ATTR_DROPOUT_SEED, torch.tensor(seed, dtype=torch.int64, device="cuda:0"))
    pd = a.moe_combine_backward.primitive_desc(
        gpu[0], c.bind(a.ARG_DIFF_DST, dy), c.grouped(a.ARG_SRC, rows, offsets), c.bind(a.ARG_SRC_1, dpos),
        c.bind(a.ARG_WEIGHTS, torch.from_numpy(weights).cuda()), c.grouped(a.ARG_DIFF_SRC, drows, offsets),
        c.bind(a.ARG_DIFF_WEIGHTS, dw), dropout_p=p)
    c.run(a.moe_combine_backward, pd).strm.wait()
    g = host(dy)
    if p:
        g = R.dropout(g, p, *seed)
    x = host(rows)
    want, want_dw, size = np.zeros_like(x), np.zeros((T, k)), np.zeros((T, k))
    for t in range(T):
        for j in range(k):
            if pos[t, j] >= 0:
                want[pos[t, j]] = weights[t, j].astype(np.float64) * g[t]
                want_dw[t, j] = (g[t] * x[pos[t, j]]).sum()
                size[t, j] = np.abs(g[t] * x[pos[t, j]]).sum()
    check(host(drows), want, np.abs(want) * 3 * EPS + out_slack(want, dtype))
    check(host(dw), want_dw, size * EPS * (H + 16) + 2.0 ** -140)


def test_combine_backward_against_differences(gpu):
    """<drows, v> + <dw, u> equals the difference of the 64-bit forward along (v, u), with dropout's mask fixed; the forward
    is bilinear, so the central difference is exact up to 64-bit rounding"""
    import torch
    r = rng(21)
    T, E, k, H, p, seed, h = 9, 8, 3, 70, 0.3, (123456789012345, 42), 1e-3
    rows, offsets, dpos, pos = make_rows(r, T, E, k, H, "f32", 0.1)
    w = r.random((T, k)).astype(np.float32)
    dy = device_matrix(r.standard_normal((T, H)), "f32")
    c = Call(gpu[0])
    a = c.api
    drows, dw = torch.empty_like(rows), torch.empty((T, k), device="cuda:0")
    c.bind(a.ARG_ATTR_DROPOUT_SEED, torch.tensor(seed, dtype=torch.int64, device="cuda:0"))
    pd = a.moe_combine_backward.primitive_desc(
        gpu[0], c.bind(a.ARG_DIFF_DST, dy), c.grouped(a.ARG_SRC, rows, offsets), c.bind(a.ARG_SRC_1, dpos),
        c.bind(a.ARG_WEIGHTS, torch.from_numpy(w).cuda()), c.grouped(a.ARG_DIFF_SRC, drows, offsets),
        c.bind(a.ARG_DIFF_WEIGHTS, dw), dropout_p=p)
    c.run(a.moe_combine_backward, pd).strm.wait()
    x, v, u = host(rows), r.standard_normal(rows.shape), r.standard_normal((T, k))

    def f(s):
        picked = np.where(pos[:, :, None] >= 0, (x + s * v)[np.maximum(pos, 0)], 0.0)
        return (R.dropout(((w.astype(np.float64) + s * u)[:, :, None] * picked).sum(1), p, *seed) * host(dy)).sum()
    got = (host(drows) * v).sum() + (host(dw) * u).sum()
    size = np.abs(host(drows) * v).sum() + np.abs(x).max() * H * np.abs(host(dy)).max() * np.abs(u).sum()
    assert abs(got - (f(h) - f(-h)) / (2 * h)) <= size * EPS * (H + 16) + 1e-9


def test_combine_inverts_dispatch(gpu):
    """rows sorted and summed back: each token times the number of its choices that got a row - dispatch's gradient"""
    r = rng(9)
    x = device_matrix(r.integers(-8, 8, (999, 72)).astype(np.float64), "bf16")
    idx = choices(r, 999, 12, 4, 0.3)
    rows, offsets, pos = run_dispatch(gpu[0], x, idx, 12)
    y = run_combine(gpu[0], rows, offsets, pos, "bf16")
    assert np.array_equal(y, host(x) * (host(pos) >= 0).sum(1, keepdims=True))


@pytest.mark.parametrize("T", [0, 3])
def test_combine_of_nothing(gpu, T):
    import torch
    H = 0 if T else 16
    rows = torch.zeros((T * 2, H), device="cuda:0")
    offsets = torch.full((4,), 2 * T, dtype=torch.int32, device="cuda:0")
    pos = torch.arange(2 * T, dtype=torch.int32, device="cuda:0").view(T, 2)
    assert run_combine(gpu[0], rows, offsets, pos, "f32").shape == (T, H)
    c = Call(gpu[0])
    a = c.api
    dw = torch.full((T, 2), 7.0, device="cuda:0")
    pd = a.moe_combine_backward.primitive_desc(
        gpu[0], c.bind(a.ARG_DIFF_DST, torch.zeros((T, H), device="cuda:0")), c.grouped(a.ARG_SRC, rows, offsets), c.bind(a.ARG_SRC_1, pos),
        c.bind(a.ARG_WEIGHTS, torch.ones((T, 2), device="cuda:0")), c.grouped(a.ARG_DIFF_SRC, torch.zeros_like(rows), offsets),
        c.bind(a.ARG_DIFF_WEIGHTS, dw))
    c.run(a.moe_combine_backward, pd).strm.wait()
    assert not host(dw).any()


def test_positions_outside_the_rows_are_skipped(gpu):
    import torch
    rows = torch.ones((8, 40), device="cuda:0")
    offsets = torch.tensor([8], dtype=torch.int32, device="cuda:0")
    pos = torch.tensor([[0, 8], [2 ** 31 - 1, -2 ** 31], [3, -1], [7, 7]], dtype=torch.int32, device="cuda:0")
    assert run_combine(gpu[0], rows, offsets, pos, "f32")[:, 0].tolist() == [1, 0, 1, 2]


@pytest.mark.parametrize("T,H,p", [(40, 104, 0.2), (40, 103, 0.2), (3000, 1024, 0.2), (3000, 1024, 0.0), (600, 4096, 0.5)])
def test_inputs_of_one_row_for_all_and_results_in_place(gpu, T, H, p):
    """residual, weights, tokens and the gradient with a row pitch of 0; dst in the residual's memory"""
    import torch
    r = rng(T, H)
    E, k, seed = 8, 2, (99, 5)
    rows, offsets, dpos, pos = make_rows(r, T, E, k, H, "bf16", 0.1)
    one, w1 = device_matrix(r.standard_normal((1, H)), "bf16"), r.random((1, k)).astype(np.float32)
    weights = torch.from_numpy(w1).cuda().expand(T, k)
    drop = dict(p=p, seed=seed if p else None)
    got = run_combine(gpu[0], rows, offsets, dpos, "bf16", weights, one.expand(T, H), **drop)
    want, size = combine_want(rows, pos, np.where(pos >= 0, w1, 0).astype(np.float64), np.repeat(host(one), T, 0), p, seed)
    check(got, want, size * EPS * (k + 4) + out_slack(want, "bf16"))
    y = device_matrix(np.repeat(host(one), T, 0), "bf16")
    c = Call(gpu[0])
    a = c.api
    if p:
        c.bind(a.ARG_ATTR_DROPOUT_SEED, torch.tensor(seed, dtype=torch.int64, device="cuda:0"))
    pd = a.moe_combine.primitive_desc(gpu[0], c.grouped(a.ARG_SRC, rows, offsets), c.bind(a.ARG_SRC_1, dpos), c.bind(a.ARG_DST, y),
                                      weights_md=c.bind(a.ARG_WEIGHTS, weights), residual_md=c.bind(a.ARG_SRC_2, y), dropout_p=p)
    c.run(a.moe_combine, pd).strm.wait()
    assert np.array_equal(host(y), got)
    c = Call(gpu[0])
    drows, dw = torch.empty_like(rows), torch.empty((T, k), device="cuda:0")
    if p:
        c.bind(a.ARG_ATTR_DROPOUT_SEED, torch.tensor(seed, dtype=torch.int64, device="cuda:0"))
    pd = a.moe_combine_backward.primitive_desc(
        gpu[0], c.bind(a.ARG_DIFF_DST, one.expand(T, H)), c.grouped(a.ARG_SRC, rows, offsets), c.bind(a.ARG_SRC_1, dpos),
        c.bind(a.ARG_WEIGHTS, weights), c.grouped(a.ARG_DIFF_SRC, drows, offsets), c.bind(a.ARG_DIFF_WEIGHTS, dw), dropout_p=p)
    c.run(a.moe_combine_backward, pd).strm.wait()
    g = np.repeat(host(one), T, 0)
    g = R.dropout(g, p, *seed) if p else g
    x = host(rows)
    dots = np.where(pos >= 0, np.einsum("th,tkh->tk", g, x[np.maximum(pos, 0)]), 0.0)
    sizes = np.einsum("th,tkh->tk", np.abs(g), np.abs(x[np.maximum(pos, 0)]))
    check(host(dw), dots, sizes * EPS * (H + 16) + 2.0 ** -140)
    idx = choices(r, T, E, k, 0)
    got_rows, _, got_pos = run_dispatch(gpu[0], one.expand(T, H), idx, E)
    assert np.array_equal(host(got_rows), np.repeat(host(one), T * k, 0)) and np.array_equal(host(got_pos), R.sort_slots(idx, E)[1])


# ----------------------------------------------------------------------------------------------- dropout


def run_dropout(eng, x, p, seed, residual=None, out=None, pitch=0):
    import torch
    c = Call(eng)
    a = c.api
    y = out if out is not None else device_matrix(np.full(tuple(x.shape), 7.0), c.name(x), pitch)
    c.bind(a.ARG_ATTR_DROPOUT_SEED, torch.tensor(seed, dtype=torch.int64, device="cuda:0"))
    pd = a.dropout.primitive_desc(eng, c.bind(a.ARG_SRC, x), c.bind(a.ARG_DST, y), p, residual_md=c.bind(a.ARG_SRC_2, residual))
    c.run(a.dropout, pd).strm.wait()
    return host(y)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("M,N,p,res,pitch,out_pitch,offset", [
    (1, 1, 0.5, False, 0, 0, 0), (1, 8191, 0.1, True, 0, 0, 0), (33, 129, 0.3, True, 0, 0, 0), (64, 4096, 0.1, True, 0, 0, 0),
    (64, 4096, 0.1, False, 4104, 4112, 0), (17, 1003, 0.25, True, 1011, 1007, 3), (301, 6, 0.9, False, 7, 0, 1), (40, 36, 0.5, True, 40, 48, 0),
    (5, 77, 0.0, True, 0, 0, 0), (5, 77, 1.0, True, 80, 0, 0), (2000, 2, 0.2, False, 3, 0, 0), (9, 4100, 0.2, True, 0, 4104, 0)])
def test_dropout(gpu, M, N, p, res, pitch, out_pitch, offset, dtype):
    r = rng(M, N, dtype)
    x = device_matrix(r.standard_normal((M, N)), dtype, pitch, offset)
    residual = device_matrix(r.standard_normal((M, N)), dtype) if res else None
    seed = (int(r.integers(0, 2 ** 62)), int(r.integers(-2 ** 62, 2 ** 62)))
    got = run_dropout(gpu[0], x, p, seed, residual, pitch=out_pitch)
    want = R.dropout(host(x), p, *seed)
    size = np.abs(want)
    if res:
        want, size = want + host(residual), size + np.abs(host(residual))
    check(got, want, size * 3 * EPS + out_slack(want, dtype))
    if not res and 0 < p < 1:  # exactly the generator's mask
        assert np.array_equal(got != 0, R.keep_mask((M, N), p, *seed)[0])


def test_dropped_elements_are_zero_whatever_they_are(gpu):
    import torch
    x = torch.full((16, 100), float("inf"), device="cuda:0")
    x[::2] = float("nan")
    keep, _ = R.keep_mask((16, 100), 0.5, 1, 2)
    got = run_dropout(gpu[0], x, 0.5, (1, 2))
    assert not got[~keep].any() and not np.isfinite(got[keep]).any()
    assert not run_dropout(gpu[0], x, 1.0, (1, 2)).any()


def test_dropout_in_place_and_its_gradient(gpu):
    """dst may be src; the gradient is the same primitive on the gradient: <D(x), g> = <x, D(g)>"""
    r = rng(3)
    x, g = (device_matrix(r.integers(-8, 8, (130, 24)).astype(np.float64), "f32") for _ in range(2))
    y, d = run_dropout(gpu[0], x, 0.5, (77, 3)), run_dropout(gpu[0], g, 0.5, (77, 3))
    assert (y * host(g)).sum() == (host(x) * d).sum()
    before = host(x)
    assert np.array_equal(run_dropout(gpu[0], x, 0.5, (77, 3), residual=x, out=x), y + before)


def test_dropout_rate(gpu):
    """the share of kept elements of 2^22: within five standard deviations of 1 - p"""
    import torch
    n = 1 << 22
    for p in (0.1, 0.37, 0.9):
        kept = (run_dropout(gpu[0], torch.ones((1, n), device="cuda:0"), p, (5, int(p * 100))) != 0).mean()
        assert abs(kept - (1 - p)) < 5 * (p * (1 - p) / n) ** 0.5


# ------------------------------------------------------------------------------------- how they are called


def test_open_dims_serve_batches_of_any_size(gpu):
    """one primitive for every number of tokens; what disagrees with the descriptor is refused"""
    import torch
    from onednn_b200 import api as a
    eng = gpu[0]
    E, k, H, O = 12, 3, 40, a.RUNTIME_DIM_VAL
    md = a.memory.desc
    prims = {}
    prims["route"] = a.moe_route(a.moe_route.primitive_desc(eng, md((O, E), 3, (E, 1)), md((O, k), 3, (k, 1)), md((O, k), 4, (k, 1))))
    prims["dispatch"] = a.moe_dispatch(a.moe_dispatch.primitive_desc(
        eng, md((O, H), 3, (H, 1)), md((O, k), 4, (k, 1)), md.grouped((O, H), 3, 0, E), md((O, k), 4, (k, 1))))
    prims["combine"] = a.moe_combine(a.moe_combine.primitive_desc(
        eng, md.grouped((O, H), 3, 0, E), md((O, k), 4, (k, 1)), md((O, H), 3, (H, 1)), weights_md=md((O, k), 3, (k, 1))))
    for T in (1, 50, 1200, 0, 7):
        r = rng(T)
        x, logits = device_matrix(r.standard_normal((T, H)), "f32"), device_matrix(r.standard_normal((T, E)), "f32")
        w, idx, pos = (torch.empty((T, k), device="cuda:0", dtype=d) for d in (torch.float32, torch.int32, torch.int32))
        rows, offsets, y = torch.empty((T * k, H), device="cuda:0"), torch.empty((E,), device="cuda:0", dtype=torch.int32), torch.empty_like(x)
        c = Call(eng)
        for name, tensors in (("route", ((a.ARG_SRC, logits), (a.ARG_DST, w), (a.ARG_DST_1, idx))),
                              ("dispatch", ((a.ARG_SRC, x), (a.ARG_SRC_1, idx), (a.ARG_DST_1, pos))),
                              ("combine", ((a.ARG_SRC_1, pos), (a.ARG_WEIGHTS, w), (a.ARG_DST, y)))):
            c.args = {}
            for arg, t in tensors:
                c.bind(arg, t)
            if name != "route":
                c.grouped(a.ARG_DST if name == "dispatch" else a.ARG_SRC, rows, offsets)
            prims[name].execute(c.strm, c.args)
        c.strm.wait()
        want_idx = R.choose(host(logits), k)
        assert np.array_equal(host(idx), want_idx)
        assert np.array_equal(host(offsets), R.sort_slots(want_idx, E)[0])
        check(host(y), host(x) * host(w).sum(1, keepdims=True), np.abs(host(x)) * EPS * 8)  # the weights sum to one
        if T == 50:  # the descriptors of one call have to agree
            c.args = {}
            for arg, t in ((a.ARG_SRC, logits), (a.ARG_DST, w[:49]), (a.ARG_DST_1, idx)):
                c.bind(arg, t)
            with pytest.raises(a.error) as e:
                prims["route"].execute(c.strm, c.args)
            assert e.value.status == a.invalid_arguments


def test_seed_is_read_on_the_device(gpu):
    """a captured graph with another seed makes another mask; a stream of the caller's own"""
    import torch
    from onednn_b200 import api as a
    x, y = torch.ones((64, 64), device="cuda:0"), torch.zeros((64, 64), device="cuda:0")
    seed = torch.tensor([1, 0], dtype=torch.int64, device="cuda:0")
    s = torch.cuda.Stream()
    c = Call(gpu[0], s.cuda_stream)
    c.bind(a.ARG_ATTR_DROPOUT_SEED, seed)
    prim = a.dropout(a.dropout.primitive_desc(gpu[0], c.bind(a.ARG_SRC, x), c.bind(a.ARG_DST, y), 0.5))
    prim.execute(c.strm, c.args)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        prim.execute(c.strm, c.args)
    for step in range(3):
        seed[1] = step
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(host(y) != 0, R.keep_mask((64, 64), 0.5, 1, step)[0])


@pytest.mark.parametrize("mode", ["library", "user"])
def test_scratchpad_modes(gpu, mode):
    import torch
    from onednn_b200 import api as a
    r = rng(8)
    T, E, k, H = 1500, 24, 3, 16
    x, idx = device_matrix(r.standard_normal((T, H)), "f32"), choices(r, T, E, k, 0)
    c = Call(gpu[0])
    rows, offsets = torch.empty((T * k, H), device="cuda:0"), torch.empty((E,), device="cuda:0", dtype=torch.int32)
    pos = torch.empty((T, k), device="cuda:0", dtype=torch.int32)
    attr = a.primitive_attr()
    attr.set_scratchpad_mode(a.SCRATCHPAD_MODE_USER if mode == "user" else a.SCRATCHPAD_MODE_LIBRARY)
    pd = a.moe_dispatch.primitive_desc(gpu[0], c.bind(a.ARG_SRC, x), c.bind(a.ARG_SRC_1, torch.from_numpy(idx).cuda()),
                                       c.grouped(a.ARG_DST, rows, offsets), c.bind(a.ARG_DST_1, pos), attr=attr)
    prim = a.moe_dispatch(pd)
    if mode == "user":
        with pytest.raises(a.error) as e:
            prim.execute(c.strm, c.args)
        assert e.value.status == a.invalid_arguments
        md = pd.query_md(136)
        c.args[a.ARG_SCRATCHPAD] = a.memory(md, gpu[0], torch.full((md.get_size(),), 255, dtype=torch.uint8, device="cuda:0").data_ptr())
    prim.execute(c.strm, c.args)
    c.strm.wait()
    ends, want_pos, _ = R.sort_slots(idx, E)
    assert np.array_equal(host(offsets), ends) and np.array_equal(host(pos), want_pos)


def test_two_runs_give_the_same_bits(gpu):
    import torch
    r = rng(13)
    rows, offsets, dpos, pos = make_rows(r, 400, 16, 4, 513, "bf16", 0.1)
    w = torch.from_numpy(r.random((400, 4)).astype(np.float32)).cuda()
    runs = [run_combine(gpu[0], rows, offsets, dpos, "f32", w, None, 0.1, (3, 4)) for _ in range(2)]
    assert np.array_equal(*runs)


def test_rows_beyond_32_bit_offsets(gpu):
    """grouped rows of more than 2^31 elements: dispatch writes and combine reads behind that"""
    import torch
    T, E, k, H = 70001, 16, 8, 4096
    r = rng(1)
    idx = r.integers(0, E, (T, k)).astype(np.int32)
    x = torch.randint(-8, 8, (T, H), device="cuda:0", dtype=torch.int8).to(torch.bfloat16)
    rows, offsets, pos = run_dispatch(gpu[0], x, idx, E)
    ends, want_pos, order = R.sort_slots(idx, E)
    assert np.array_equal(host(offsets), ends) and np.array_equal(host(pos), want_pos)
    at = np.array([0, 1, T * k // 2, 2 ** 31 // H, T * k - 1])
    assert torch.equal(rows[torch.from_numpy(at).cuda()], x[torch.from_numpy(order[at] // k).cuda()])
    c = Call(gpu[0])
    a = c.api
    y = torch.empty_like(x)
    pd = a.moe_combine.primitive_desc(gpu[0], c.grouped(a.ARG_SRC, rows, offsets), c.bind(a.ARG_SRC_1, pos), c.bind(a.ARG_DST, y))
    c.run(a.moe_combine, pd).strm.wait()
    assert torch.equal(y, x * k)


@pytest.mark.parametrize("tokens,dropout", [(512, 0.1), (1, 0.0), (37, 0.0), (1300, 0.3)])
def test_a_layer_of_all_of_them(gpu, tokens, dropout):
    """router, dispatch, the experts' products, combine and the gradients in one stream, each reading what the one before
    wrote (examples/moe_layer.py).  The sums of 2048 bf16 products round to 8 bits on the way (2^-8 of a row's size, a row's
    largest values being a few times its usual ones): 2 % of the largest result."""
    import os
    import sys
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
    import moe_layer
    difference, layer = moe_layer.run(tokens=tokens, dropout=dropout)
    assert max(difference.values()) < 0.02, difference
    want = R.choose(host(layer.logits), 4)
    assert np.array_equal(host(layer.idx), want)
    assert np.array_equal(host(layer.offsets), R.sort_slots(want, 16)[0])

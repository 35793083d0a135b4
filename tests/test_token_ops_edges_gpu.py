"""The operators around an expert layer's products, and dropout: contents, sizes and uses at their edges, against plain 64-bit
forms.  Every input is made from fixed numbers.  Tolerances as in test_token_ops_gpu.py."""
import zlib

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


# ----------------------------------------------------------------------------------------------- combine


def run_combine_backward(eng, rows, offsets, pos, weights, dy, p=0.0, seed=None):
    """gradients of the rows and of the weights, in memory that holds other values before"""
    import torch
    c = base.Call(eng)
    a = c.api
    drows, dw = torch.full_like(rows, 7.0), torch.full(tuple(pos.shape), 7.0, device="cuda:0")
    if p:
        c.bind(a.ARG_ATTR_DROPOUT_SEED, torch.tensor(seed, dtype=torch.int64, device="cuda:0"))
    pd = a.moe_combine_backward.primitive_desc(
        eng, c.bind(a.ARG_DIFF_DST, dy), c.grouped(a.ARG_SRC, rows, offsets), c.bind(a.ARG_SRC_1, pos), c.bind(a.ARG_WEIGHTS, weights),
        c.grouped(a.ARG_DIFF_SRC, drows, offsets), c.bind(a.ARG_DIFF_WEIGHTS, dw), dropout_p=p)
    c.run(a.moe_combine_backward, pd).strm.wait()
    return host(drows), host(dw)


def check_both_ways(eng, r, rows, offsets, pos, p):
    """combine and its gradient for the positions in `pos`, those outside the groups' rows naming nothing"""
    import torch
    T, k = pos.shape
    H, dtype, kept = rows.shape[1], base.Call(eng).name(rows), int(offsets[-1])
    named = (pos >= 0) & (pos < kept)
    at = np.where(named, pos, -1)
    weights = r.standard_normal((T, k)).astype(np.float32)
    dpos, dweights = torch.from_numpy(pos).cuda(), torch.from_numpy(weights).cuda()
    seed = (int(r.integers(0, 2 ** 62)), int(r.integers(0, 2 ** 62))) if p else None
    got = base.run_combine(eng, rows, offsets, dpos, dtype, dweights, None, p, seed)
    want, size = base.combine_want(rows, at, np.where(named, weights, 0).astype(np.float64), None, p, seed)
    base.check(got, want, size * EPS * (k + 4) + out_slack(want, dtype))
    dy = device_matrix(r.standard_normal((T, H)), dtype)
    drows, dw = run_combine_backward(eng, rows, offsets, dpos, dweights, dy, p, seed)
    g = R.dropout(host(dy), p, *seed) if p else host(dy)
    x, slots = host(rows), np.argwhere(named)
    where = pos[named]
    want, want_dw, size = np.zeros_like(x), np.zeros((T, k)), np.zeros((T, k))
    want[where] = weights[named].astype(np.float64)[:, None] * g[slots[:, 0]]
    terms = g[slots[:, 0]] * x[where]
    want_dw[named], size[named] = terms.sum(1), np.abs(terms).sum(1)
    base.check(drows, want, np.abs(want) * 3 * EPS + np.where(want != 0, out_slack(want, dtype), 0))
    base.check(dw, want_dw, size * EPS * (H + 16) + np.where(named, 2.0 ** -140, 0))


FORMS = [  # a warp and a CTA a token, rows on and off 16-byte boundaries, few and many choices, and the ring of bulk copies
    (37, 8, 2, 104, "bf16", 0.0), (300, 64, 8, 2048, "bf16", 0.2), (300, 12, 3, 2047, "f16", 0.0), (64, 6, 4, 7, "f32", 0.25),
    (150, 40, 32, 520, "f32", 0.0), (2101, 16, 3, 1032, "bf16", 0.0), (2050, 16, 8, 1024, "bf16", 0.2)]


@pytest.mark.parametrize("T,E,k,H,dtype,p", FORMS)
def test_positions_behind_the_last_group_name_nothing(gpu, T, E, k, H, dtype, p):
    """the rows behind the last offset belong to no slot: forward leaves them out, backward zeroes them, whoever names them"""
    import torch
    r = rng(T, E, k, H)
    rows, offsets, _, pos = base.make_rows(r, T, E, k, H, dtype, 0.3)
    kept = int(offsets[-1])
    assert kept < T * k
    out = np.argwhere(pos < 0)
    behind = out[r.random(len(out)) < 0.6]
    pos[behind[:, 0], behind[:, 1]] = r.integers(kept, T * k, len(behind))
    check_both_ways(gpu[0], r, rows, offsets, pos, p)


@pytest.mark.parametrize("dtype,H", [("f32", 40), ("bf16", 41)])
def test_offsets_beyond_the_memory_are_cut(gpu, dtype, H):
    """a last offset above the number of rows, or below zero"""
    import torch
    r = rng(H)
    rows, offsets, dpos, pos = base.make_rows(r, 20, 5, 2, H, dtype, 0)
    for last, there in ((2 ** 31 - 1, 1.0), (-5, 0.0)):
        offsets[-1] = last
        y = base.run_combine(gpu[0], rows, offsets, dpos, "f32")
        base.check(y, there * host(rows)[pos].sum(1), np.abs(host(rows)[pos]).sum(1) * EPS * 8)
        drows, dw = run_combine_backward(gpu[0], rows, offsets, dpos, torch.ones((20, 2), device="cuda:0"),
                                         device_matrix(np.ones((20, H)), dtype))
        assert (drows == there).all() and (dw != 0).all() == bool(there)


@pytest.mark.parametrize("T,E,k,H,dtype,p", FORMS + [(9000, 64, 4, 16, "bf16", 0.0), (70001, 8, 4, 8, "f32", 0.0)])
def test_rows_whose_slots_were_taken_back_have_no_gradient(gpu, T, E, k, H, dtype, p):
    """positions a program set to -1 after dispatch (tokens over an expert's capacity): the rows stay in their groups, and
    what the groups' products make of their gradient counts; it is zero"""
    r = rng(T, E, k, H, 1)
    rows, offsets, _, pos = base.make_rows(r, T, E, k, H, dtype, 0.1)
    taken = r.random(pos.shape) < 0.3
    taken[T // 2] = True
    taken[:, 0] |= pos[:, 0] < r.integers(0, 40)  # whole words of rows
    pos[taken] = -1
    check_both_ways(gpu[0], r, rows, offsets, pos, p)


@pytest.mark.parametrize("T,k,pitch,offset", [(3000, 3, 5, 1), (2000, 8, 8, 1), (41, 4, 9, 0)])
def test_positions_inside_a_wider_buffer(gpu, T, k, pitch, offset):
    r = rng(T, k)
    rows, offsets, _, pos = base.make_rows(r, T, 11, k, 72, "bf16", 0.1)
    pos[r.random(pos.shape) < 0.2] = -1
    dpos = device_matrix(pos, "s32", pitch, offset)
    w, dy = device_matrix(r.standard_normal((T, k)), "f32", pitch, offset), device_matrix(r.standard_normal((T, 72)), "bf16")
    drows, dw = run_combine_backward(gpu[0], rows, offsets, dpos, w, dy)
    named = pos >= 0
    want, g = np.zeros(tuple(rows.shape)), host(dy)
    want[pos[named]] = host(w)[named][:, None] * g[np.argwhere(named)[:, 0]]
    base.check(drows, want, np.abs(want) * 3 * EPS + np.where(want != 0, out_slack(want, "bf16"), 0))
    assert not dw[~named].any() and dw[named].all()


def test_no_slot_names_a_row(gpu):
    r = rng(2)
    rows, offsets, _, pos = base.make_rows(r, 700, 6, 2, 264, "bf16", 0)
    pos[:] = -1
    check_both_ways(gpu[0], r, rows, offsets, pos, 0.0)


# (the ring of bulk copies at its limits: one row a token, as few and as many as it takes, several tokens an item, ragged ones)
RING = [(4100, 8, 1, 4104, "bf16", "bf16", 0.2), (2049, 8, 1, 8200, "f32", "f16", 0.0), (2100, 16, 3, 1000, "f32", "f32", 0.3),
        (2051, 16, 12, 1032, "bf16", "f32", 0.1), (701, 16, 12, 3080, "f32", "f32", 0.0), (2063, 16, 7, 1040, "f16", "f16", 0.0),
        (1500, 40, 13, 1544, "bf16", "bf16", 0.1), (1400, 40, 32, 1544, "f32", "bf16", 0.0), (4099, 8, 2, 2056, "bf16", "bf16", 0.3),
        (4100, 8, 2, 8200, "bf16", "bf16", 0.1)]


@pytest.mark.parametrize("T,E,k,H,dtype,out,p", RING)
def test_combine_on_both_sides_of_the_ring(gpu, T, E, k, H, dtype, out, p):
    base.test_combine(gpu, T, E, k, H, dtype, out, True, k % 2 == 1, p, 0, 0.05)


# ---------------------------------------------------------------------------------------------- dispatch


def guarded(shape, dtype, value):
    """a tensor in the middle of a buffer, and a check that nothing around it changed"""
    import torch
    n, pad = int(np.prod(shape)), 4096
    buf = torch.full((n + 2 * pad,), value, dtype=dtype, device="cuda:0")

    def untouched():
        return bool((buf[:pad] == value).all() and (buf[pad + n:] == value).all())
    return buf[pad:pad + n].view(shape), untouched


@pytest.mark.parametrize("H", [64, 65])  # both copies
def test_one_dispatch_on_two_streams_with_scratchpads_of_their_own(gpu, H):
    """one primitive in flight twice, above the number of slots from which counts go through the scratchpad; nothing is
    written around the outputs and the scratchpads"""
    import torch
    from onednn_b200 import api as a
    eng, T, E, k = gpu[0], 6000, 48, 3
    attr = a.primitive_attr()
    attr.set_scratchpad_mode(a.SCRATCHPAD_MODE_USER)
    prim, calls = None, []
    for n in range(2):
        r = rng(H, n)
        x, idx = device_matrix(r.standard_normal((T, H)), "bf16"), base.choices(r, T, E, k, 0.1)
        c = base.Call(eng, torch.cuda.Stream().cuda_stream)
        rows, rows_ok = guarded((T * k, H), torch.bfloat16, 7)
        offsets, offsets_ok = guarded((E,), torch.int32, 7)
        pos, pos_ok = guarded((T, k), torch.int32, 7)
        mds = [c.bind(a.ARG_SRC, x), c.bind(a.ARG_SRC_1, torch.from_numpy(idx).cuda()), c.grouped(a.ARG_DST, rows, offsets),
               c.bind(a.ARG_DST_1, pos)]
        if prim is None:
            pd = a.moe_dispatch.primitive_desc(eng, *mds, attr=attr)
            prim = a.moe_dispatch(pd)
        md = pd.query_md(136)
        assert md.get_size() > 0
        scratch, scratch_ok = guarded((md.get_size(),), torch.uint8, 255)
        c.args[a.ARG_SCRATCHPAD] = a.memory(md, eng, scratch.data_ptr())
        calls.append((c, x, idx, rows, offsets, pos, scratch, (rows_ok, offsets_ok, pos_ok, scratch_ok)))
    torch.cuda.synchronize()
    for _ in range(20):
        for call in calls:
            prim.execute(call[0].strm, call[0].args)
    torch.cuda.synchronize()
    for c, x, idx, rows, offsets, pos, scratch, checks in calls:
        ends, want_pos, order = R.sort_slots(idx, E)
        want = np.zeros((T * k, H))
        want[:order.size] = host(x)[order // k]
        assert np.array_equal(host(offsets), ends) and np.array_equal(host(pos), want_pos) and np.array_equal(host(rows), want)
        assert all(ok() for ok in checks) and not (scratch == 255).all()


@pytest.mark.parametrize("T,E,k,H,dtype,pitch", [(128, 8, 2, 4096, "bf16", 0), (100, 5, 2, 1001, "f16", 1004), (60, 7, 4, 5003, "s8", 0),
                                                     (96, 8, 2, 8192, "bf16", 0), (60, 5, 2, 2001, "f16", 2004), (24, 9, 8, 5003, "s8", 0)])
def test_few_slots_of_wide_rows(gpu, T, E, k, H, dtype, pitch):
    """the form of one launch, rows wide enough that its grid goes round"""
    r = rng(T, H)
    x = device_matrix(r.integers(-100, 100, (T, H)).astype(np.float64), dtype, pitch)
    idx = base.choices(r, T, E, k, 0.1)
    rows, offsets, pos = base.run_dispatch(gpu[0], x, idx, E)
    ends, want_pos, order = R.sort_slots(idx, E)
    want = np.zeros((T * k, H))
    want[:order.size] = host(x)[order // k]
    assert np.array_equal(host(offsets), ends) and np.array_equal(host(pos), want_pos) and np.array_equal(host(rows), want)


@pytest.mark.parametrize("mode", ["library", "user"])
def test_scratchpad_of_many_slots(gpu, mode):
    """above the number of slots from which counts go through the scratchpad; a user's holds other values before every call"""
    import torch
    from onednn_b200 import api as a
    r = rng(12)
    T, E, k, H = 4000, 24, 3, 16
    attr = a.primitive_attr()
    attr.set_scratchpad_mode(a.SCRATCHPAD_MODE_USER if mode == "user" else a.SCRATCHPAD_MODE_LIBRARY)
    x, idx = device_matrix(r.standard_normal((T, H)), "f32"), base.choices(r, T, E, k, 0.1)
    c = base.Call(gpu[0])
    rows, offsets = torch.empty((T * k, H), device="cuda:0"), torch.empty((E,), device="cuda:0", dtype=torch.int32)
    pos, didx = torch.empty((T, k), device="cuda:0", dtype=torch.int32), torch.from_numpy(idx).cuda()
    pd = a.moe_dispatch.primitive_desc(gpu[0], c.bind(a.ARG_SRC, x), c.bind(a.ARG_SRC_1, didx), c.grouped(a.ARG_DST, rows, offsets),
                                       c.bind(a.ARG_DST_1, pos), attr=attr)
    prim, md, untouched = a.moe_dispatch(pd), pd.query_md(136), lambda: True
    assert (md.get_ndims() > 0) == (mode == "user")
    if mode == "user":
        with pytest.raises(a.error) as e:
            prim.execute(c.strm, c.args)
        assert e.value.status == a.invalid_arguments
        scratch, untouched = guarded((md.get_size(),), torch.uint8, 255)
        c.args[a.ARG_SCRATCHPAD] = a.memory(md, gpu[0], scratch.data_ptr())
    for n in range(3):
        if n:
            idx = base.choices(r, T, E, k, 0.3)
            didx.copy_(torch.from_numpy(idx))
            if mode == "user":
                scratch.fill_(255 if n == 1 else 1)
        torch.cuda.synchronize()
        prim.execute(c.strm, c.args)
        c.strm.wait()
        ends, want_pos, order = R.sort_slots(idx, E)
        assert np.array_equal(host(offsets), ends) and np.array_equal(host(pos), want_pos)
        assert np.array_equal(host(rows)[:order.size], host(x)[order // k]) and untouched()
    if mode == "user":
        assert not (scratch == 1).all()


# ----------------------------------------------------------------------------------------------- dropout


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("M,N,p,res,pitch", [
    (1, 3 * 148 * 4 * 4096 + 4101, 0.1, True, 0), (1, 2 * 148 * 4 * 4096 + 3, 0.5, False, 0), (2600, 2048, 0.2, True, 2056),
    (1700, 3076, 0.3, False, 3080), (4099, 1367, 0.25, True, 1371), (9001, 255, 0.1, False, 0), (1200, 2001, 1.0, True, 2003),
    (1500, 1024, 1.0, False, 0)])
def test_dropout_of_tensors_that_outnumber_the_grid(gpu, M, N, p, res, pitch, dtype):
    """every form whose grid stays goes round at least once: one long row, aligned rows, rows that start anywhere, p = 1"""
    r = rng(M, N)
    x = device_matrix(r.standard_normal((M, N), dtype=np.float32), dtype, pitch)
    residual = device_matrix(r.standard_normal((M, N), dtype=np.float32), dtype) if res else None
    seed = (int(r.integers(0, 2 ** 62)), int(r.integers(0, 2 ** 62)))
    got = base.run_dropout(gpu[0], x, p, seed, residual, pitch=pitch)
    want = R.dropout(host(x), p, *seed)
    size = np.abs(want)
    if res:
        want, size = want + host(residual), size + np.abs(host(residual))
    base.check(got, want, size * 3 * EPS + out_slack(want, dtype))


# ------------------------------------------------------------------------------------- how they are called


def test_one_dispatch_of_open_dims_for_batches_on_both_sides_of_its_forms(gpu):
    """few slots, slots that every CTA counts, and slots counted through the scratchpad, in turn"""
    import torch
    from onednn_b200 import api as a
    eng, E, k, H, O = gpu[0], 30, 4, 24, a.RUNTIME_DIM_VAL
    md, prim = a.memory.desc, None
    for T in (5000, 17, 9000, 1500, 2100, 0, 30001):
        r = rng(T)
        x, idx = device_matrix(r.integers(-100, 100, (T, H)).astype(np.float64), "f32"), base.choices(r, T, E, k, 0.1)
        c = base.Call(eng)
        rows, offsets = torch.full((T * k, H), 7.0, device="cuda:0"), torch.full((E,), 7, device="cuda:0", dtype=torch.int32)
        pos = torch.full((T, k), 7, device="cuda:0", dtype=torch.int32)
        mds = [c.bind(a.ARG_SRC, x, (0,)), c.bind(a.ARG_SRC_1, torch.from_numpy(idx).cuda(), (0,)),
               c.grouped(a.ARG_DST, rows, offsets, open_rows=True), c.bind(a.ARG_DST_1, pos, (0,))]
        if prim is None:
            prim = a.moe_dispatch(a.moe_dispatch.primitive_desc(eng, *mds))
        prim.execute(c.strm, c.args)
        c.strm.wait()
        ends, want_pos, order = R.sort_slots(idx, E)
        assert np.array_equal(host(offsets), ends) and np.array_equal(host(pos), want_pos)
        assert np.array_equal(host(rows)[:order.size], host(x)[order // k]) and not host(rows)[order.size:].any()


def test_gradients_and_dropout_of_open_dims(gpu):
    """one primitive of each for batches of any size; memory that contradicts the rest is refused"""
    import torch
    from onednn_b200 import api as a
    eng, E, k, H, p, seed = gpu[0], 12, 3, 40, 0.3, (77, 5)
    prims = {}
    dseed = torch.tensor(seed, dtype=torch.int64, device="cuda:0")
    for T in (50, 1, 1200, 0, 7):
        r = rng(T, 9)
        # the router's gradient
        logits, g = device_matrix(r.standard_normal((T, E)), "f32"), r.standard_normal((T, k)).astype(np.float32)
        idx, d = R.choose(host(logits), k), torch.full((T, E), 7.0, device="cuda:0")
        c = base.Call(eng)
        mds = [c.bind(arg, t, (0,)) for arg, t in ((a.ARG_SRC, logits), (a.ARG_SRC_1, torch.from_numpy(idx).cuda()),
                                                  (a.ARG_DIFF_DST, torch.from_numpy(g).cuda()), (a.ARG_DIFF_SRC, d))]
        if "route" not in prims:
            prims["route"] = a.moe_route_backward(a.moe_route_backward.primitive_desc(eng, *mds))
        prims["route"].execute(c.strm, c.args)
        c.strm.wait()
        want, size = R.route_backward(host(logits), idx, g.astype(np.float64), "softmax", True, 1.0)
        spread = np.ptp(host(logits)) if T else 0
        base.check(host(d), want, size * EPS * (4 * (2 + spread) + 64 + k) + out_slack(want, "f32") + 2.0 ** -140)
        # combine's
        rows, offsets, dpos, pos = base.make_rows(r, T, E, k, H, "bf16", 0.1)
        w, dy = r.standard_normal((T, k)).astype(np.float32), device_matrix(r.standard_normal((T, H)), "bf16")
        drows, dw = torch.full_like(rows, 7.0), torch.full((T, k), 7.0, device="cuda:0")
        c = base.Call(eng)
        c.bind(a.ARG_ATTR_DROPOUT_SEED, dseed)
        mds = [c.bind(a.ARG_DIFF_DST, dy, (0, 1)), c.grouped(a.ARG_SRC, rows, offsets, open_rows=True), c.bind(a.ARG_SRC_1, dpos, (0,)),
               c.bind(a.ARG_WEIGHTS, torch.from_numpy(w).cuda(), (0,)), c.grouped(a.ARG_DIFF_SRC, drows, offsets, open_rows=True),
               c.bind(a.ARG_DIFF_WEIGHTS, dw, (0, 1))]
        if "combine" not in prims:
            prims["combine"] = a.moe_combine_backward(a.moe_combine_backward.primitive_desc(eng, *mds, dropout_p=p))
        prims["combine"].execute(c.strm, c.args)
        c.strm.wait()
        gy, x, named = R.dropout(host(dy), p, *seed), host(rows), pos >= 0
        want, want_dw, size = np.zeros_like(x), np.zeros((T, k)), np.zeros((T, k))
        slots, where = np.argwhere(named), pos[named]
        want[where] = w[named].astype(np.float64)[:, None] * gy[slots[:, 0]]
        want_dw[named], size[named] = (gy[slots[:, 0]] * x[where]).sum(1), np.abs(gy[slots[:, 0]] * x[where]).sum(1)
        base.check(host(drows), want, np.abs(want) * 3 * EPS + out_slack(want, "bf16"))
        base.check(host(dw), want_dw, size * EPS * (H + 16) + 2.0 ** -140)
        # dropout, with an open width too
        x = device_matrix(r.standard_normal((T, 33 + T % 5)), "f16")
        y = torch.full_like(x, 7.0)
        c = base.Call(eng)
        c.bind(a.ARG_ATTR_DROPOUT_SEED, dseed)
        mds = [c.bind(a.ARG_SRC, x, (0, 1)), c.bind(a.ARG_DST, y, (0, 1)), c.bind(a.ARG_SRC_2, x, (0, 1))]
        if "dropout" not in prims:
            prims["dropout"] = a.dropout(a.dropout.primitive_desc(eng, mds[0], mds[1], p, residual_md=mds[2]))
        prims["dropout"].execute(c.strm, c.args)
        c.strm.wait()
        kept = R.dropout(host(x), p, *seed)
        base.check(host(y), kept + host(x), (np.abs(kept) + np.abs(host(x))) * 3 * EPS + out_slack(kept + host(x), "f16"))
        if T == 50:
            c.bind(a.ARG_DST, y[:49])
            with pytest.raises(a.error) as e:
                prims["dropout"].execute(c.strm, c.args)
            assert e.value.status == a.invalid_arguments


# ------------------------------------------------------------- tests of test_token_ops_gpu.py with inputs that stay


@pytest.fixture
def fixed(monkeypatch):
    """(the module draws its inputs from hash() of a string, which every process salts anew)"""
    monkeypatch.setattr(base, "rng", lambda *key: rng(*(zlib.crc32(k.encode()) if isinstance(k, str) else k for k in key)))


@pytest.mark.parametrize("scoring,normalize", base.MODES)
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("T,E,k", base.SHAPES)
def test_route_with_fixed_inputs(gpu, fixed, T, E, k, dtype, scoring, normalize):
    base.test_route(gpu, T, E, k, dtype, scoring, normalize)
    base.test_route_backward(gpu, T, E, k, dtype, scoring, normalize)


DROPOUTS = next(m.args[1] for m in base.test_dropout.pytestmark if m.args[0].startswith("M,N"))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("M,N,p,res,pitch,out_pitch,offset", DROPOUTS)
def test_dropout_with_fixed_inputs(gpu, fixed, M, N, p, res, pitch, out_pitch, offset, dtype):
    base.test_dropout(gpu, M, N, p, res, pitch, out_pitch, offset, dtype)

"""The root-mean-square norm, its 8-bit outputs and its gradient on a device, against 64-bit forms (layer_ref.py)."""
import numpy as np
import pytest

import layer_ref as L
import token_ref as R

pytestmark = pytest.mark.gpu

EPSILON = 1e-5
# every number of threads and chunks that a row can have, odd widths, single columns
WIDTHS = [1, 8, 40, 255, 256, 264, 512, 513, 1000, 1367, 2048, 2047, 4096, 4104, 8192, 8200, 16384, 16383, 5001, 7001]


def values(seed, shape, dtype, scale=1.0):
    """what `dtype` holds, as 64-bit numbers; rows of different sizes"""
    r = np.random.Generator(np.random.PCG64(seed))
    a = r.standard_normal(shape) * scale
    if len(shape) == 2:
        a *= np.exp(r.standard_normal((shape[0], 1)))
    return L.rounded(a, dtype)


def device(a, dtype, pitch=0, offset=0):
    return None if a is None else R.device_matrix(a, dtype, pitch, offset)


def vector(a, dtype, offset=0):
    return None if a is None else R.device_matrix(a[None, :], dtype, 0, offset)[0]


def empty(shape, dtype, pitch=0, offset=0):
    """a matrix inside a buffer of a known byte, and the buffer"""
    import torch
    m, n = shape
    ld = pitch or n
    size = torch.empty(0, dtype=L.torch_dtype(dtype)).element_size()
    raw = torch.full(((offset + m * ld) * size,), 0x5a, dtype=torch.uint8, device="cuda:0")
    return raw.view(L.torch_dtype(dtype))[offset:].view(m, ld)[:, :n], raw


def untouched(raw, shape, dtype, pitch=0, offset=0):
    import torch
    m, n = shape
    size = torch.empty(0, dtype=L.torch_dtype(dtype)).element_size()
    bytes_ = raw.cpu().numpy()
    assert (bytes_[:offset * size] == 0x5a).all()
    assert (bytes_[offset * size:].reshape(m, (pitch or n) * size)[:, n * size:] == 0x5a).all()


def run_norm(gpu, x, dt, out, weights=None, wdt="f32", residual=None, total=False, scaling="", group=0, given=None, pitch=0, offset=0,
             out_pitch=0, out_offset=0, epsilon=EPSILON):
    """(q or y, scales, sum) as 64-bit numbers"""
    import torch
    from onednn_b200 import api
    c = L.Call(gpu[0])
    T, H = x.shape
    dst, raw = empty((T, H), out, out_pitch, out_offset)
    sums, sums_raw = empty((T, H), dt, pitch) if total else (None, None)
    attr, scales, dynamic = None, None, dict(qmode=api.quantization_mode.dynamic_fp)
    if scaling:
        attr = api.primitive_attr()
        if scaling == "tensor":
            attr.set_scales(api.ARG_DST, 0)
            scales = torch.tensor([given], dtype=torch.float32, device="cuda:0")
        elif scaling == "row":
            attr.set_scales(api.ARG_DST, 1, **dynamic)
            scales = torch.full((T, 1), -7.0, device="cuda:0")
        else:
            attr.set_scales(api.ARG_DST, 3, (1, group), **dynamic)
            scales = torch.full((T, H // group), -7.0, device="cuda:0")
        c.bind(api.ARG_ATTR_SCALES | api.ARG_DST, scales)
    pd = api.rms_norm.primitive_desc(
        gpu[0], c.bind(api.ARG_SRC, device(x, dt, pitch, offset)), c.bind(api.ARG_DST, dst), epsilon,
        weights_md=c.bind(api.ARG_WEIGHTS, vector(weights, wdt)), residual_md=c.bind(api.ARG_SRC_2, device(residual, dt)),
        sum_md=c.bind(api.ARG_DST_1, sums), attr=attr)
    c.run(api.rms_norm, pd)
    c.strm.wait()
    untouched(raw, (T, H), out, out_pitch, out_offset)
    if total:
        untouched(sums_raw, (T, H), dt, pitch)
    return R.host(dst if out != "e4m3" else dst.float()), None if scales is None else R.host(scales), R.host(sums) if total else None


def close(got, want, units, dtype):
    with np.errstate(invalid="ignore"):
        bad = ~(np.abs(got - want) <= units * L.EPS * np.abs(want) + R.out_slack(want, dtype))
    assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], want[bad][:5])


@pytest.mark.parametrize("H", WIDTHS)
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_norm(gpu, H, dtype):
    """16 or 32 bits, the residual and the sum, each kind of weights; rows that are aligned where the width allows"""
    T = 11 if H <= 512 else 3
    x, res, w = values(H, (T, H), dtype), values(H + 1, (T, H), dtype), values(H + 2, (H,), dtype)
    got, _, total = run_norm(gpu, x, dtype, dtype, w, dtype, res, True)
    want, h = L.norm(x, EPSILON, w, res)
    close(got, want, L.NORM_UNITS, dtype)
    close(total, h, 1, dtype)
    got, _, _ = run_norm(gpu, x, dtype, "f32", values(H + 2, (H,), "f32"))
    close(got, L.norm(x, EPSILON, values(H + 2, (H,), "f32"))[0], L.NORM_UNITS, "f32")
    got, _, _ = run_norm(gpu, x, dtype, dtype)
    close(got, L.norm(x, EPSILON)[0], L.NORM_UNITS, dtype)


@pytest.mark.parametrize("T,H", [(5001, 24), (9000, 200), (4000, 520), (2500, 1000), (3001, 1367), (1500, 2048), (1300, 3000), (700, 4096), (650, 5001),
                                 (600, 5120), (500, 7001), (450, 8192)])
@pytest.mark.parametrize("dtype,residual", [("bf16", True), ("bf16", False), ("f32", True)])
def test_norm_of_many_rows(gpu, T, H, dtype, residual):
    """more rows than CTAs: each takes several, with the next on its way"""
    x, w = values(1, (T, H), dtype), values(3, (H,), "f32")
    res = values(2, (T, H), dtype) if residual else None
    got, scale, total = run_norm(gpu, x, dtype, "s8", w, residual=res, total=residual, scaling="row")
    y, h = L.norm(x, EPSILON, w, res)
    v, s = L.quantized(y, "s8", 0)
    close(scale, s, L.NORM_UNITS + 1, "f32")
    L.check_8bit(got, v, 2 * L.NORM_UNITS + 4, "s8")
    if residual:
        close(total, h, 1, dtype)
    if H % 8 == 0:
        got, _, _ = run_norm(gpu, x, dtype, dtype, w, residual=res)
        close(got, y, L.NORM_UNITS, dtype)
    if H % 128 == 0:
        got, scale, _ = run_norm(gpu, x, dtype, "e4m3", w, residual=res, scaling="group", group=128)
        v, s = L.quantized(y, "e4m3", 128)
        close(scale, s, L.NORM_UNITS + 1, "f32")
        L.check_8bit(got, v, 2 * L.NORM_UNITS + 4, "e4m3")


@pytest.mark.parametrize("pitch,offset,out_pitch,out_offset", [(0, 1, 0, 0), (1003, 0, 0, 0), (0, 0, 1001, 0), (0, 0, 0, 3),
                                                               (1008, 8, 1024, 16)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_norm_of_rows_that_start_anywhere(gpu, pitch, offset, out_pitch, out_offset, dtype):
    x, w = values(5, (5, 1000), dtype), values(6, (1000,), "f32")
    for out in (dtype, "s8", "e4m3"):
        scaling = {} if out == dtype else dict(scaling="row")
        got, scale, _ = run_norm(gpu, x, dtype, out, w, pitch=pitch, offset=offset, out_pitch=out_pitch, out_offset=out_offset, **scaling)
        y = L.norm(x, EPSILON, w)[0]
        if out == dtype:
            close(got, y, L.NORM_UNITS, dtype)
        else:
            v, s = L.quantized(y, out, 0)
            close(scale, s, L.NORM_UNITS + 1, "f32")
            L.check_8bit(got, v, 2 * L.NORM_UNITS + 4, out)


@pytest.mark.parametrize("scaling,H,group", [("tensor", 264, 0), ("tensor", 255, 0), ("row", 8, 0), ("row", 513, 0), ("row", 4096, 0),
                                             ("row", 16384, 0)]
                         + [("group", H, g) for H, g in ((16, 16), (48, 16), (96, 32), (320, 64), (640, 128), (2304, 256), (4096, 128),
                                                         (16384, 128))])
@pytest.mark.parametrize("out", ["s8", "e4m3"])
@pytest.mark.parametrize("dtype,offset", [("bf16", 0), ("f32", 0), ("f16", 1)])
def test_norm_in_8_bits(gpu, scaling, H, group, out, dtype, offset):
    T = 9 if H <= 512 else 4
    x, res, w = values(H, (T, H), dtype), values(H + 1, (T, H), dtype), values(H + 2, (H,), "f32")
    given = 2.5 / L.LIMIT[out]  # (some values saturate)
    got, scale, total = run_norm(gpu, x, dtype, out, w, residual=res, total=True, scaling=scaling, group=group, given=given, offset=offset)
    y, h = L.norm(x, EPSILON, w, res)
    close(total, h, 1, dtype)
    if scaling == "tensor":
        v = y / float(np.float32(given))
    else:
        v, s = L.quantized(y, out, group)
        close(scale, s, L.NORM_UNITS + 1, "f32")
    # y and the scale (or its reciprocal) each off by NORM_UNITS, two divisions and a product
    L.check_8bit(got, v, 2 * L.NORM_UNITS + 4, out)


@pytest.mark.parametrize("out", ["s8", "e4m3"])
def test_norm_in_8_bits_without_scales(gpu, out):
    x = values(1, (4, 64), "f32") * 1.0
    got, _, _ = run_norm(gpu, x, "f32", out, values(2, (64,), "f32", 90.0))
    L.check_8bit(got, L.norm(x, EPSILON, values(2, (64,), "f32", 90.0))[0], L.NORM_UNITS, out)


@pytest.mark.parametrize("scaling,group", [("row", 0), ("group", 32), ("tensor", 0)])
@pytest.mark.parametrize("out", ["s8", "e4m3"])
@pytest.mark.parametrize("offset", [0, 1])
def test_rows_of_zeros_infinities_and_nan(gpu, scaling, group, out, offset):
    H = 96
    x = values(3, (6, H), "f32")
    x[0] = 0
    x[1, 5] = np.nan
    x[2, 7] = np.inf
    x[3] *= 1e-30  # squares vanish beside epsilon, values do not: scales of the smallest kind
    x[4] = 0
    x[4, 40] = 2.0  # two of three groups hold zeros only
    got, scale, _ = run_norm(gpu, x, "f32", out, None, scaling=scaling, group=group, given=0.01, offset=offset)
    assert (got[0] == 0).all()
    nan_rows = got[1:3]
    if out == "e4m3":
        assert np.isnan(nan_rows[0]).all() and np.isnan(nan_rows[1, 7]) and (scaling != "row" or np.isnan(nan_rows[1]).all())
    else:
        assert (nan_rows[0] == 0).all() and nan_rows[1, 7] == 0
    if scaling != "tensor":
        assert (scale[0] == 0).all() and np.isnan(scale[1]).all() and np.isnan(scale[2]).any()
        y = L.norm(x[3:], EPSILON)[0]
        parts = y.reshape(3, -1, group or H)
        most = np.abs(parts).max(2)
        close(scale[3:], most / L.LIMIT[out], L.NORM_UNITS + 1, "f32")
        with np.errstate(invalid="ignore"):
            v = np.where(most[:, :, None] > 0, parts / (most[:, :, None] / L.LIMIT[out]), 0).reshape(3, H)
        L.check_8bit(got[3:], v, 2 * L.NORM_UNITS + 4, out)


def test_tiny_rows_have_a_scale_of_zero(gpu):
    x = np.full((2, 64), 1e-38)
    x[1] *= 300  # the largest value is 1e-36 x 316 x 3 after the norm: has a scale
    x = L.rounded(x, "f32")
    got, scale, _ = run_norm(gpu, x, "f32", "s8", None, scaling="row", epsilon=1.0)
    assert scale[0, 0] == 0 and (got[0] == 0).all()
    assert scale[1, 0] > 0 and (got[1] == 127).all()


def run_backward(gpu, h, dy, dt, weights=None, wdt="f32", dsum=None, dweights="f32", pitch=0, offset=0, epsilon=EPSILON, c=None):
    import torch
    from onednn_b200 import api
    c = c or L.Call(gpu[0])
    T, H = h.shape
    out, raw = empty((T, H), dt, pitch, offset)
    dw = torch.full((H,), 3.0, dtype=R.torch_dtype(dweights), device="cuda:0") if dweights else None
    pd = api.rms_norm_backward.primitive_desc(
        gpu[0], c.bind(api.ARG_DIFF_DST, device(dy, dt, pitch)), c.bind(api.ARG_SRC, device(h, dt, 0, offset)), c.bind(api.ARG_DIFF_SRC, out),
        epsilon, weights_md=c.bind(api.ARG_WEIGHTS, vector(weights, wdt)), diff_weights_md=c.bind(api.ARG_DIFF_WEIGHTS, dw),
        diff_sum_md=c.bind(api.ARG_SRC_2, device(dsum, dt)))
    c.run(api.rms_norm_backward, pd)
    c.strm.wait()
    untouched(raw, (T, H), dt, pitch, offset)
    return R.host(out), None if dw is None else R.host(dw)


def check_backward(got, gotw, h, dy, dt, w, dsum, dweights):
    dh, dw, size, wsize = L.norm_backward(h, dy, EPSILON, w, dsum)
    assert (np.abs(got - dh) <= L.NORM_GRAD_UNITS * L.EPS * size + R.out_slack(dh, dt)).all()
    if dweights:
        # terms off by 28 units, summed one after the other at worst
        units = 28 + h.shape[0] + 45
        assert (np.abs(gotw - dw) <= units * L.EPS * wsize + R.out_slack(dw, dweights)).all()


@pytest.mark.parametrize("H", WIDTHS)
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_backward(gpu, H, dtype):
    T = 13 if H <= 512 else 5
    h, dy, dsum = (values(H + i, (T, H), dtype) for i in range(3))
    for w, wdt, add, dweights in ((values(H + 3, (H,), dtype), dtype, dsum, "f32"), (values(H + 3, (H,), "f32"), "f32", None, dtype),
                                  (None, "f32", dsum, None)):
        got, gotw = run_backward(gpu, h, dy, dtype, w, wdt, add, dweights)
        check_backward(got, gotw, h, dy, dtype, w, add, dweights)


@pytest.mark.parametrize("T,H,pitch,offset", [(4099, 64, 0, 0), (3001, 520, 0, 0), (1300, 1367, 1371, 0), (700, 4096, 4104, 8), (5000, 37, 0, 1),
                                              (901, 2056, 2057, 0)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_backward_of_many_rows(gpu, T, H, pitch, offset, dtype):
    """more rows than CTAs: each takes several"""
    h, dy, w = values(1, (T, H), dtype), values(2, (T, H), dtype), values(3, (H,), "f32")
    got, gotw = run_backward(gpu, h, dy, dtype, w, "f32", None, "f32", pitch, offset)
    check_backward(got, gotw, h, dy, dtype, w, None, "f32")


def test_backward_against_differences(gpu):
    """the gradient that the device makes, against differences of the forward pass in 64 bits"""
    T, H = 3, 24
    h, dy, w = values(1, (T, H), "f32"), values(2, (T, H), "f32"), values(3, (H,), "f32")
    got, gotw = run_backward(gpu, h, dy, "f32", w)
    step = 1e-6
    for t in range(T):
        for i in range(H):
            up, down = h.copy(), h.copy()
            up[t, i] += step
            down[t, i] -= step
            num = ((L.norm(up, EPSILON, w)[0] - L.norm(down, EPSILON, w)[0]) * dy).sum() / (2 * step)
            assert abs(num - got[t, i]) < 2e-5 * np.abs(got).max()
    for i in range(H):
        up, down = w.copy(), w.copy()
        up[i] += step
        down[i] -= step
        num = ((L.norm(h, EPSILON, up)[0] - L.norm(h, EPSILON, down)[0]) * dy).sum() / (2 * step)
        assert abs(num - gotw[i]) < 2e-5 * np.abs(gotw).max()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_no_rows(gpu, dtype):
    import torch
    from onednn_b200 import api
    got, scale, _ = run_norm(gpu, np.zeros((0, 64)), dtype, "s8", scaling="row")
    assert got.shape == (0, 64)
    got, gotw = run_backward(gpu, np.zeros((0, 64)), np.zeros((0, 64)), dtype, np.ones(64))
    assert (gotw == 0).all()  # (they were 3)


def test_results_in_place_and_one_row_for_all(gpu):
    import torch
    from onednn_b200 import api
    T, H = 40, 512
    x, res, w = values(1, (T, H), "bf16"), values(2, (T, H), "bf16"), values(3, (H,), "f32")
    want, h = L.norm(x, EPSILON, w, res)
    c = L.Call(gpu[0])
    xt, rt, wt = device(x, "bf16"), device(res, "bf16"), vector(w, "f32")
    pd = api.rms_norm.primitive_desc(gpu[0], c.bind(api.ARG_SRC, xt), c.bind(api.ARG_DST, xt), EPSILON, weights_md=c.bind(api.ARG_WEIGHTS, wt),
                                     residual_md=c.bind(api.ARG_SRC_2, rt), sum_md=c.bind(api.ARG_DST_1, rt))
    c.run(api.rms_norm, pd)
    c.strm.wait()
    close(R.host(xt), want, L.NORM_UNITS, "bf16")
    close(R.host(rt), h, 1, "bf16")
    # a row pitch of zero: the same row every time
    c = L.Call(gpu[0])
    one, y = device(x[:1], "bf16"), torch.empty((T, H), dtype=torch.bfloat16, device="cuda:0")
    pd = api.rms_norm.primitive_desc(gpu[0], c.bind(api.ARG_SRC, one.expand(T, H)), c.bind(api.ARG_DST, y), EPSILON)
    c.run(api.rms_norm, pd)
    c.strm.wait()
    close(R.host(y), np.repeat(L.norm(x[:1], EPSILON)[0], T, 0), L.NORM_UNITS, "bf16")
    # the gradient over dy's memory
    dy = values(4, (T, H), "bf16")
    dh, dw, size, wsize = L.norm_backward(x, dy, EPSILON, w)
    c = L.Call(gpu[0])
    g = device(dy, "bf16")
    pd = api.rms_norm_backward.primitive_desc(gpu[0], c.bind(api.ARG_DIFF_DST, g), c.bind(api.ARG_SRC, device(x, "bf16")),
                                              c.bind(api.ARG_DIFF_SRC, g), EPSILON, weights_md=c.bind(api.ARG_WEIGHTS, wt))
    c.run(api.rms_norm_backward, pd)
    c.strm.wait()
    assert (np.abs(R.host(g) - dh) <= L.NORM_GRAD_UNITS * L.EPS * size + R.out_slack(dh, "bf16")).all()


def test_open_dims_serve_batches_of_any_size(gpu):
    import torch
    from onednn_b200 import api
    H, open_rows = 256, (0,)
    w = values(3, (H,), "f32")
    attr = api.primitive_attr()
    attr.set_scales(api.ARG_DST, 3, (1, 64), qmode=api.quantization_mode.dynamic_fp)
    prim = back = None
    for T in (3, 40, 0, 1):
        x, dy = values(T, (T, H), "bf16"), values(T + 1, (T, H), "bf16")
        c = L.Call(gpu[0])
        dst = torch.empty((T, H), dtype=torch.int8, device="cuda:0")
        scales = torch.empty((T, H // 64), device="cuda:0")
        mds = [c.bind(a, t, open_rows) for a, t in ((api.ARG_SRC, device(x, "bf16")), (api.ARG_DST, dst))]
        c.bind(api.ARG_ATTR_SCALES | api.ARG_DST, scales)
        wmd = c.bind(api.ARG_WEIGHTS, vector(w, "f32"))
        prim = prim or api.rms_norm(api.rms_norm.primitive_desc(gpu[0], *mds, EPSILON, weights_md=wmd, attr=attr))
        prim.execute(c.strm, c.args)
        c.strm.wait()
        if T:
            v, s = L.quantized(L.norm(x, EPSILON, w)[0], "s8", 64)
            close(R.host(scales), s, L.NORM_UNITS + 1, "f32")
            L.check_8bit(R.host(dst), v, 2 * L.NORM_UNITS + 4, "s8")
        small = torch.empty((max(T - 1, 0), H // 64), device="cuda:0")
        if T:
            c.bind(api.ARG_ATTR_SCALES | api.ARG_DST, small)
            with pytest.raises(api.error) as e:
                prim.execute(c.strm, c.args)
            assert e.value.status == api.invalid_arguments
        c = L.Call(gpu[0])
        out, dw = torch.empty((T, H), dtype=torch.bfloat16, device="cuda:0"), torch.empty(H, device="cuda:0")
        mds = [c.bind(a, t, open_rows) for a, t in ((api.ARG_DIFF_DST, device(dy, "bf16")), (api.ARG_SRC, device(x, "bf16")),
                                                    (api.ARG_DIFF_SRC, out))]
        wmd, dwmd = c.bind(api.ARG_WEIGHTS, vector(w, "f32")), c.bind(api.ARG_DIFF_WEIGHTS, dw)
        back = back or api.rms_norm_backward(api.rms_norm_backward.primitive_desc(gpu[0], *mds, EPSILON, weights_md=wmd, diff_weights_md=dwmd))
        back.execute(c.strm, c.args)
        c.strm.wait()
        check_backward(R.host(out), R.host(dw), x, dy, "bf16", w, None, "f32")


def test_captured_and_replayed_on_another_stream(gpu):
    """forward and backward in one graph, its inputs changed between replays; each graph with a scratchpad of its own"""
    import torch
    from onednn_b200 import api
    T, H = 64, 1024
    s = torch.cuda.Stream()
    x, dy, w = (torch.empty(sh, dtype=torch.bfloat16, device="cuda:0") for sh in ((T, H), (T, H), (H,)))
    y, dh, dw = torch.empty_like(x), torch.empty_like(x), torch.empty(H, device="cuda:0")
    attr = api.primitive_attr()
    attr.set_scratchpad_mode(api.SCRATCHPAD_MODE_USER)
    f, b = L.Call(gpu[0], s.cuda_stream), L.Call(gpu[0], s.cuda_stream)
    fpd = api.rms_norm.primitive_desc(gpu[0], f.bind(api.ARG_SRC, x), f.bind(api.ARG_DST, y), EPSILON, weights_md=f.bind(api.ARG_WEIGHTS, w))
    bpd = api.rms_norm_backward.primitive_desc(gpu[0], b.bind(api.ARG_DIFF_DST, dy), b.bind(api.ARG_SRC, x), b.bind(api.ARG_DIFF_SRC, dh), EPSILON,
                                               weights_md=b.bind(api.ARG_WEIGHTS, w), diff_weights_md=b.bind(api.ARG_DIFF_WEIGHTS, dw), attr=attr)
    need = bpd.query_md(255, api.ARG_SCRATCHPAD).get_dims()[0]
    b.bind(api.ARG_SCRATCHPAD, torch.empty(need, dtype=torch.uint8, device="cuda:0"))
    fp, bp = api.rms_norm(fpd), api.rms_norm_backward(bpd)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        fp.execute(f.strm, f.args)
        bp.execute(b.strm, b.args)
    for seed in (1, 2):
        a, g, ww = values(seed, (T, H), "bf16"), values(seed + 10, (T, H), "bf16"), values(seed + 20, (H,), "bf16")
        for t, v in ((x, a), (dy, g), (w, ww)):
            t.copy_(torch.from_numpy(v))
        graph.replay()
        torch.cuda.synchronize()
        close(R.host(y), L.norm(a, EPSILON, ww)[0], L.NORM_UNITS, "bf16")
        check_backward(R.host(dh), R.host(dw), a, g, "bf16", ww, None, "f32")


def test_two_runs_give_the_same_bits(gpu):
    h, dy, w = values(1, (3000, 1024), "bf16"), values(2, (3000, 1024), "bf16"), values(3, (1024,), "f32")
    a, b = (run_backward(gpu, h, dy, "bf16", w) for _ in range(2))
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


def test_rows_beyond_32_bit_offsets(gpu):
    """a buffer of more than 2^32 elements: the last row's place needs 64 bits"""
    import torch
    from onednn_b200 import api
    H, T, pitch = 64, 5, (1 << 30) + 64
    buf = torch.empty((T - 1) * pitch + H, dtype=torch.bfloat16, device="cuda:0")
    x = torch.as_strided(buf, (T, H), (pitch, 1))
    a = values(1, (T, H), "bf16")
    x.copy_(torch.from_numpy(a))
    c = L.Call(gpu[0])
    c.run(api.rms_norm, api.rms_norm.primitive_desc(gpu[0], c.bind(api.ARG_SRC, x), c.bind(api.ARG_DST, x), EPSILON))
    c.strm.wait()
    close(R.host(x), L.norm(a, EPSILON)[0], L.NORM_UNITS, "bf16")


@pytest.mark.parametrize("out", ["s8", "e4m3"])
def test_the_norm_feeds_a_quantized_product(gpu, out):
    """norm -> 8 bits with scales -> dnnl::matmul, which takes the scales that the norm wrote (s8) or was given (e4m3)"""
    import torch
    from onednn_b200 import api
    T, H, N = 96, 1024, 256
    x, w = values(1, (T, H), "bf16"), values(2, (H,), "f32")
    r = np.random.Generator(np.random.PCG64(9))
    wei = r.integers(-127, 128, (H, N)) if out == "s8" else L.rounded(r.standard_normal((H, N)), "e4m3")
    wscale = L.rounded(r.random(N) + 0.5, "f32")
    c = L.Call(gpu[0])
    q = torch.empty((T, H), dtype=L.torch_dtype(out), device="cuda:0")
    attr, mattr = api.primitive_attr(), api.primitive_attr()
    if out == "s8":
        attr.set_scales(api.ARG_DST, 1, qmode=api.quantization_mode.dynamic_fp)
        mattr.set_scales(api.ARG_SRC, 1)
        scales = torch.empty((T, 1), device="cuda:0")
    else:
        attr.set_scales(api.ARG_DST, 0)
        mattr.set_scales(api.ARG_SRC, 0)
        scales = torch.tensor([0.01], device="cuda:0")
    mattr.set_scales(api.ARG_WEIGHTS, 2)
    c.bind(api.ARG_ATTR_SCALES | api.ARG_DST, scales)
    pd = api.rms_norm.primitive_desc(gpu[0], c.bind(api.ARG_SRC, device(x, "bf16")), c.bind(api.ARG_DST, q), EPSILON,
                                     weights_md=c.bind(api.ARG_WEIGHTS, vector(w, "f32")), attr=attr)
    m = L.Call(gpu[0])
    wt = torch.from_numpy(np.ascontiguousarray(wei)).to("cuda:0").to(L.torch_dtype(out))
    dst = torch.empty((T, N), device="cuda:0")
    m.bind(api.ARG_ATTR_SCALES | api.ARG_SRC, scales)
    m.bind(api.ARG_ATTR_SCALES | api.ARG_WEIGHTS, vector(wscale, "f32"))
    mpd = api.matmul.primitive_desc(gpu[0], m.bind(api.ARG_SRC, q), m.bind(api.ARG_WEIGHTS, wt), m.bind(api.ARG_DST, dst), None, mattr)
    assert mpd.impl_info_str() == {"s8": "cuda:tcgen05:int8", "e4m3": "cuda:tcgen05:fp8"}[out]
    c.run(api.rms_norm, pd)
    m.run(api.matmul, mpd)
    m.strm.wait()
    qv = R.host(q.float())
    want = (qv @ wei) * R.host(scales).reshape(-1, 1) * wscale
    size = (np.abs(qv) @ np.abs(wei)) * R.host(scales).reshape(-1, 1) * wscale
    assert (np.abs(R.host(dst) - want) <= 4 * L.EPS * np.abs(want) + 4 * L.EPS * size).all()
    # and from the unquantized product by no more than each operand's rounding (half a step, or what saturation cut off) times
    # its weight; the scales' and the product's own 32-bit errors come on top
    y, s = L.norm(x, EPSILON, w)[0], R.host(scales).reshape(-1, 1)
    v = np.clip(y / s, -L.LIMIT[out], L.LIMIT[out])
    off = np.abs(y / s - v) + (0.5 if out == "s8" else L.step_e4m3(v) / 2) + 2 * (2 * L.NORM_UNITS + 4) * L.EPS * np.abs(v)
    assert (np.abs(R.host(dst) - (y @ wei) * wscale) <= (off @ np.abs(wei)) * s * wscale + 8 * L.EPS * size).all()

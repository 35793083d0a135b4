"""Low-rank adapters on a device, against 64-bit forms (layer_ref.py)."""
import numpy as np
import pytest

import layer_ref as L
import token_ref as R

pytestmark = pytest.mark.gpu


def rng(*seed):
    return np.random.Generator(np.random.PCG64([sum(map(ord, str(s))) for s in seed]))


def factor(a, dtype, layout, offset=0):
    """[n, p, q] on the device with neighbours along q ("last"), along p ("middle"), or every stride above one ("wide")"""
    import torch
    n, p, q = a.shape
    buf = torch.zeros(offset + 2 * a.size + 8, dtype=R.torch_dtype(dtype), device="cuda:0")[offset:]
    strides = {"last": (p * q, q, 1), "middle": (p * q, 1, p), "wide": (2 * p * q, 2 * q, 2)}[layout]
    t = torch.as_strided(buf, (n, p, q), strides, buf.storage_offset())
    t.copy_(torch.from_numpy(np.ascontiguousarray(a)))
    return t


def run(gpu, x, index, down, up, dtype, out, scale=None, base=None, down_layout="last", up_layout="last", pitch=0, offset=0, weight_offset=0,
        in_place=False, c=None):
    import torch
    from onednn_b200 import api
    c = c or L.Call(gpu[0])
    T, N = x.shape[0], up.shape[2]
    ld = N + pitch
    raw = torch.full((T * ld + 4,), 7.0, dtype=R.torch_dtype(out), device="cuda:0")
    dst = raw[:T * ld].view(T, ld)[:, :N]
    b = None
    if base is not None:
        if in_place:
            dst.copy_(torch.from_numpy(base))
            b = dst
        else:
            b = R.device_matrix(base, out)
    attr = None
    if scale is not None:
        attr = api.primitive_attr()
        attr.set_scales(api.ARG_WEIGHTS, 1)
        c.bind(api.ARG_ATTR_SCALES | api.ARG_WEIGHTS, R.device_matrix(scale[None], "f32")[0])
    pd = api.low_rank_adapter.primitive_desc(
        gpu[0], c.bind(api.ARG_SRC, R.device_matrix(x, dtype, x.shape[1] + pitch if pitch else 0, offset)),
        c.bind(api.ARG_SRC_1, torch.from_numpy(index.astype(np.int32)).cuda()), c.bind(api.ARG_WEIGHTS, factor(down, dtype, down_layout, weight_offset)),
        c.bind(api.ARG_WEIGHTS_1, factor(up, dtype, up_layout, weight_offset)), c.bind(api.ARG_DST, dst), base_md=c.bind(api.ARG_SRC_2, b), attr=attr)
    c.run(api.low_rank_adapter, pd)
    c.strm.wait()
    rest = R.host(raw)
    assert (rest[T * ld:] == 7).all() and (rest[:T * ld].reshape(T, ld)[:, N:] == 7).all()
    return R.host(dst)


def make(T, n, K, r, N, dtype, seed=0, none=0.15, order="mixed"):
    g = rng(T, n, K, r, N, seed)
    x = L.rounded(g.standard_normal((T, K)), dtype)
    down = L.rounded(g.standard_normal((n, K, r)) * max(K, 1) ** -0.5, dtype)
    up = L.rounded(g.standard_normal((n, r, N)) * r ** -0.5, dtype)
    index = g.integers(0, n, T)
    if order == "sorted":
        index = np.sort(index)
    index[g.random(T) < none] = -1
    return x, index, down, up, L.rounded(g.random(n) + 0.5, "f32"), g


def verify(got, x, index, down, up, scale, base, dtype, out):
    y, second, both = L.low_rank(x, index, down, up, scale, base)
    bound = L.low_rank_bound(y, second, both, base, x.shape[1], down.shape[2], dtype, out)
    bad = ~(np.abs(got - y) <= bound)
    assert not bad.any(), (bad.sum(), np.argwhere(bad)[:5], got[bad][:5], y[bad][:5], bound[bad][:5])


# rows, adapters, columns in, rank, columns out: one row; ranks on both sides of every block; widths that are no multiple of
# anything; more rows than a window; tiles that are full, ragged, of one row
SIZES = [(1, 1, 64, 8, 64), (1, 5, 4096, 16, 4096), (3, 2, 8, 4, 8), (17, 2, 520, 16, 264), (64, 3, 256, 32, 128), (65, 1, 256, 24, 200), (130, 4, 192, 64, 96),
         (100, 3, 136, 128, 72), (33, 2, 64, 100, 40), (61, 64, 1024, 16, 1024), (513, 7, 128, 8, 136), (1100, 40, 64, 12, 64), (600, 1, 72, 32, 80),
         # both sides of what one launch serves, more rows than the scratchpad holds at a time, as many adapters as there can be
         (1024, 5, 64, 16, 72), (1025, 5, 64, 32, 72), (512, 3, 96, 64, 136), (513, 3, 96, 33, 136), (1200, 2, 96, 128, 136), (8300, 5, 64, 8, 72),
         (1300, 1024, 64, 16, 64), (700, 1024, 64, 16, 64)]
ODD = [(1100, 3, 33, 5, 41), (600, 2, 70, 77, 50), (1, 1, 1, 1, 1), (5, 2, 31, 3, 17), (40, 3, 1001, 16, 333), (70, 2, 40, 5, 99), (20, 2, 257, 33, 129), (9, 2, 77, 127, 55), (530, 9, 63, 7, 65)]


@pytest.mark.parametrize("T,n,K,r,N", SIZES)
@pytest.mark.parametrize("dtype,out", [("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32")])
@pytest.mark.parametrize("layouts", [("last", "last"), ("middle", "middle"), ("middle", "last"), ("last", "middle")])
def test_adapters(gpu, T, n, K, r, N, dtype, out, layouts):
    x, index, down, up, scale, g = make(T, n, K, r, N, dtype)
    base = L.rounded(g.standard_normal((T, N)), out)
    got = run(gpu, x, index, down, up, dtype, out, scale, base, *layouts)
    verify(got, x, index, down, up, scale, base, dtype, out)
    assert np.array_equal(got[index < 0], base[index < 0])


@pytest.mark.parametrize("T,n,K,r,N", ODD)
@pytest.mark.parametrize("dtype,out", [("bf16", "bf16"), ("f16", "f32")])
@pytest.mark.parametrize("layouts", [("last", "middle"), ("middle", "last"), ("wide", "wide")])
def test_odd_sizes(gpu, T, n, K, r, N, dtype, out, layouts):
    x, index, down, up, scale, g = make(T, n, K, r, N, dtype)
    got = run(gpu, x, index, down, up, dtype, out, scale, None, *layouts)
    verify(got, x, index, down, up, scale, None, dtype, out)
    assert (got[index < 0] == 0).all()


@pytest.mark.parametrize("pitch,offset,weight_offset", [(8, 8, 8), (5, 0, 0), (0, 1, 0), (0, 0, 1), (0, 0, 2), (0, 0, 4), (3, 3, 3)])
@pytest.mark.parametrize("r", [8, 32, 64])
@pytest.mark.parametrize("layouts", [("last", "last"), ("middle", "middle")])
def test_strides_and_alignment(gpu, pitch, offset, weight_offset, r, layouts):
    x, index, down, up, scale, g = make(50, 3, 128, r, 160, "bf16")
    base = L.rounded(g.standard_normal((50, 160)), "bf16")
    got = run(gpu, x, index, down, up, "bf16", "bf16", None, base, *layouts, pitch, offset, weight_offset)
    verify(got, x, index, down, up, None, base, "bf16", "bf16")


@pytest.mark.parametrize("order", ["sorted", "mixed"])
@pytest.mark.parametrize("T", [2, 15, 16, 63, 129, 511, 512, 1025])
def test_lengths_and_orders(gpu, T, order):
    x, index, down, up, scale, g = make(T, 6, 96, 16, 104, "bf16", order=order)
    base = L.rounded(g.standard_normal((T, 104)), "bf16")
    got = run(gpu, x, index, down, up, "bf16", "bf16", scale, base, "middle", "middle")
    verify(got, x, index, down, up, scale, base, "bf16", "bf16")


def test_in_place_and_rows_without_an_adapter(gpu):
    T, N = 200, 264
    x, index, down, up, scale, g = make(T, 4, 128, 16, N, "bf16")
    index[::7] = [4, -1, 1 << 30, -(1 << 31), 5, 99, -2][0]
    index[3], index[10], index[17] = -(1 << 31), (1 << 31) - 1, 4
    base = L.rounded(g.standard_normal((T, N)), "bf16")
    got = run(gpu, x, index, down, up, "bf16", "bf16", scale, base, in_place=True)
    verify(got, x, index, down, up, scale, base, "bf16", "bf16")
    none = np.full(T, -1)
    assert np.array_equal(run(gpu, x, none, down, up, "bf16", "bf16", scale, base, in_place=True), base)
    assert np.array_equal(run(gpu, x, none, down, up, "bf16", "bf16", scale, base), base)
    assert (run(gpu, x, none, down, up, "bf16", "bf16") == 0).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("out", ["same", "f32"])
def test_sizes_of_values(gpu, dtype, out):
    """middle products beyond what 16 bits hold, and far below; infinities and NaN stay in their rows"""
    out = dtype if out == "same" else out
    T, n, K, r, N = 12, 2, 64, 8, 40
    x, index, down, up, scale, g = make(T, n, K, r, N, dtype, none=0)
    big = 6e4 if dtype == "f16" else 1e30
    x[0] *= big / 8  # f16: middle products of some 10^5
    x[1] *= 1e-4
    down[:, :, 3] *= 1e-2
    up *= 1e-3
    x, down, up = L.rounded(x, dtype), L.rounded(down, dtype), L.rounded(up, dtype)
    x[4, 5], x[6, 6], x[7, :] = np.inf, np.nan, 0
    if dtype == "f16":
        x[0] = np.clip(x[0], -big, big)
    got = run(gpu, x, index, down, up, dtype, "f32" if dtype == "bf16" else out, scale, None)
    clean = [i for i in range(T) if i not in (4, 6)]
    o = "f32" if dtype == "bf16" else out
    verify(got[clean], x[clean], index[clean], down, up, scale, None, dtype, o)
    assert not np.isfinite(got[4]).any() and np.isnan(got[6]).all() and (got[7] == 0).all()


def test_long_rows(gpu):
    """every CTA of a cluster goes round its loops"""
    x, index, down, up, scale, g = make(70, 2, 16384, 16, 16384, "bf16")
    base = L.rounded(g.standard_normal((70, 16384)), "bf16")
    got = run(gpu, x, index, down, up, "bf16", "bf16", scale, base, "middle", "middle")
    verify(got, x, index, down, up, scale, base, "bf16", "bf16")


@pytest.mark.parametrize("T,K,N", [(0, 64, 64), (5, 0, 64), (5, 64, 0)])
def test_nothing(gpu, T, K, N):
    g = rng(1)
    x, index = np.zeros((T, K)), np.zeros(T, int)
    base = L.rounded(g.standard_normal((T, N)), "bf16")
    got = run(gpu, x, index, np.zeros((2, K, 8)), np.ones((2, 8, N)), "bf16", "bf16", None, base)
    assert np.array_equal(got, base)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_gradient_of_the_rows(gpu, dtype):
    """the same primitive with the factors transposed and exchanged: <dx, v> is the directional difference of <y, g>"""
    import torch
    T, n, K, r, N = 90, 5, 160, 16, 224
    x, index, down, up, scale, g = make(T, n, K, r, N, dtype)
    gy, dbase = L.rounded(g.standard_normal((T, N)), dtype), L.rounded(g.standard_normal((T, K)), dtype)
    got = run(gpu, gy, index, up.transpose(0, 2, 1), down.transpose(0, 2, 1), dtype, dtype, scale, dbase, "middle", "middle")
    verify(got, gy, index, up.transpose(0, 2, 1), down.transpose(0, 2, 1), scale, dbase, dtype, dtype)
    v = g.standard_normal((T, K))
    f = [(L.low_rank(x + s * v, index, down, up, scale)[0] * gy).sum() for s in (0.5, -0.5)]  # (linear: any step)
    _, second, both = L.low_rank(gy, index, up.transpose(0, 2, 1), down.transpose(0, 2, 1), scale)
    bound = L.low_rank_bound(got, second, both, dbase, N, r, dtype, dtype)
    assert abs(((got - dbase) * v).sum() - (f[0] - f[1])) <= (bound * np.abs(v)).sum()


def test_open_dims_and_a_captured_graph(gpu):
    import torch
    from onednn_b200 import api
    n, K, r, N = 5, 128, 16, 192
    attr = api.primitive_attr()
    attr.set_scales(api.ARG_WEIGHTS, 1)
    prim = None

    def call(T, stream=None):
        x, index, down, up, scale, g = make(T, n, K, r, N, "bf16", T)
        c = L.Call(gpu[0], stream)
        t = dict(x=R.device_matrix(x, "bf16"), i=torch.from_numpy(index.astype(np.int32)).cuda(), d=factor(down, "bf16", "middle"),
                 u=factor(up, "bf16", "middle"), y=torch.empty((T, N), dtype=torch.bfloat16, device="cuda:0"))
        mds = [c.bind(api.ARG_SRC, t["x"], (0,)), c.bind(api.ARG_SRC_1, t["i"]), c.bind(api.ARG_WEIGHTS, t["d"]), c.bind(api.ARG_WEIGHTS_1, t["u"]),
               c.bind(api.ARG_DST, t["y"], (0,))]
        mds[1] = api.memory.desc((api.RUNTIME_DIM_VAL,), 4, (1,))
        c.bind(api.ARG_ATTR_SCALES | api.ARG_WEIGHTS, R.device_matrix(scale[None], "f32")[0])
        return c, mds, t, (x, index, down, up, scale)

    for T in (1, 700, 0, 33):
        c, mds, t, a = call(T)
        prim = prim or api.low_rank_adapter(api.low_rank_adapter.primitive_desc(gpu[0], *mds, attr=attr))
        prim.execute(c.strm, c.args)
        c.strm.wait()
        verify(R.host(t["y"]), *a, None, "bf16", "bf16")
    s = torch.cuda.Stream()
    c, _, t, a = call(40, s.cuda_stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        prim.execute(c.strm, c.args)
    for shift in (0, 1):  # other rows, other adapters for them
        index = np.roll(a[1], shift)
        t["i"].copy_(torch.from_numpy(index.astype(np.int32)))
        t["y"].zero_()
        graph.replay()
        torch.cuda.synchronize()
        verify(R.host(t["y"]), a[0], index, *a[2:], None, "bf16", "bf16")


@pytest.mark.parametrize("T,out", [(1500, "bf16"), (1500, "f32"), (300, "bf16")])
def test_in_place_with_a_scratchpad_of_the_program(gpu, T, out):
    import torch
    from onednn_b200 import api
    n, K, r, N = 4, 128, 16, 200
    x, index, down, up, scale, g = make(T, n, K, r, N, "bf16", none=0.3)
    base = L.rounded(g.standard_normal((T, N)), out)
    attr = api.primitive_attr()
    attr.set_scales(api.ARG_WEIGHTS, 1)
    attr.set_scratchpad_mode(api.SCRATCHPAD_MODE_USER)
    c = L.Call(gpu[0])
    y = R.device_matrix(base, out)
    c.bind(api.ARG_ATTR_SCALES | api.ARG_WEIGHTS, R.device_matrix(scale[None], "f32")[0])
    ymd = c.bind(api.ARG_DST, y)
    c.bind(api.ARG_SRC_2, y)
    pd = api.low_rank_adapter.primitive_desc(
        gpu[0], c.bind(api.ARG_SRC, R.device_matrix(x, "bf16")), c.bind(api.ARG_SRC_1, torch.from_numpy(index.astype(np.int32)).cuda()),
        c.bind(api.ARG_WEIGHTS, factor(down, "bf16", "middle")), c.bind(api.ARG_WEIGHTS_1, factor(up, "bf16", "last")), ymd, base_md=ymd, attr=attr)
    md = pd.query_md(255, api.ARG_SCRATCHPAD)
    if T <= 512:
        assert md.get_ndims() == 0
    else:
        prim, need = api.low_rank_adapter(pd), md.get_dims()[0]
        with pytest.raises(api.error) as e:
            prim.execute(c.strm, c.args)  # none
        assert e.value.status == api.invalid_arguments
        room = torch.full((need + 32,), 0xff, dtype=torch.uint8, device="cuda:0")
        c.bind(api.ARG_SCRATCHPAD, room[4:4 + need])  # not on a 16-byte boundary
        with pytest.raises(api.error) as e:
            prim.execute(c.strm, c.args)
        assert e.value.status == api.invalid_arguments
        c.bind(api.ARG_SCRATCHPAD, room[:need])
    c.run(api.low_rank_adapter, pd)
    c.strm.wait()
    verify(R.host(y), x, index, down, up, scale, base, "bf16", out)
    assert np.array_equal(R.host(y)[index < 0], base[index < 0])


def test_calls_in_a_row(gpu):
    """each call's rows are what the call before wrote, with no wait in between: kernels that start early read behind their wait"""
    import torch
    from onednn_b200 import api
    T, n, K, r = 1400, 3, 256, 16
    x, index, down, up, scale, g = make(T, n, K, r, K, "bf16")
    a, b = R.device_matrix(x, "bf16"), torch.zeros((T, K), dtype=torch.bfloat16, device="cuda:0")
    i, d, u = torch.from_numpy(index.astype(np.int32)).cuda(), factor(down, "bf16", "middle"), factor(up, "bf16", "middle")
    calls = []
    for step in range(6):
        src, dst = (a, b) if step % 2 == 0 else (b, a)
        c = L.Call(gpu[0])
        pd = api.low_rank_adapter.primitive_desc(gpu[0], c.bind(api.ARG_SRC, src), c.bind(api.ARG_SRC_1, i), c.bind(api.ARG_WEIGHTS, d),
                                                 c.bind(api.ARG_WEIGHTS_1, u), c.bind(api.ARG_DST, dst), base_md=c.bind(api.ARG_SRC_2, src))
        calls.append((api.low_rank_adapter(pd), c))
    torch.cuda.synchronize()
    for prim, c in calls:
        prim.execute(c.strm, c.args)
    c.strm.wait()
    got = R.host(a)
    a.copy_(torch.from_numpy(x))  # the same, one at a time
    for prim, c in calls:
        prim.execute(c.strm, c.args)
        c.strm.wait()
    assert np.array_equal(got, R.host(a))


def test_two_runs_give_the_same_bits_and_a_row_does_not_depend_on_its_neighbours(gpu):
    x, index, down, up, scale, g = make(300, 6, 512, 16, 256, "bf16")
    a = run(gpu, x, index, down, up, "bf16", "f32", scale, None)
    b = run(gpu, x, index, down, up, "bf16", "f32", scale, None)
    assert np.array_equal(a, b)


def test_rows_and_adapters_beyond_32_bit_offsets(gpu):
    import torch
    from onednn_b200 import api
    T, n, K, r, N = 3, 3, 64, 8, 64
    x, index, down, up, scale, g = make(T, n, K, r, N, "bf16", none=0)
    index[:] = [2, 0, 2]
    far = (1 << 31) + 64
    c = L.Call(gpu[0])
    big = torch.empty(2 * far + 16384, dtype=torch.bfloat16, device="cuda:0")
    xs, ys = torch.as_strided(big, (T, K), (far, 1)), torch.as_strided(big, (T, N), (far, 1), 1024)
    ds, us = torch.as_strided(big, (n, K, r), (far, r, 1), 4096), torch.as_strided(big, (n, r, N), (far, N, 1), 8192)
    big = None
    for t, v in ((xs, x), (ds, down), (us, up)):
        t.copy_(torch.from_numpy(v))
    pd = api.low_rank_adapter.primitive_desc(gpu[0], c.bind(api.ARG_SRC, xs), c.bind(api.ARG_SRC_1, torch.from_numpy(index.astype(np.int32)).cuda()),
                                             c.bind(api.ARG_WEIGHTS, ds), c.bind(api.ARG_WEIGHTS_1, us), c.bind(api.ARG_DST, ys))
    c.run(api.low_rank_adapter, pd)
    c.strm.wait()
    verify(R.host(ys), x, index, down, up, None, None, "bf16", "bf16")

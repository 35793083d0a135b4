"""The norm on a device where values are special: ties of the 8-bit rounding, magnitudes at both ends of 32 bits."""
import numpy as np
import pytest

import layer_ref as L
from test_norm_gpu import check_backward, close, run_backward, run_norm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,offset", [("f32", 0), ("bf16", 0), ("bf16", 1)])
def test_rows_whose_squares_exceed_32_bits_are_zeros(gpu, dtype, offset):
    """whatever the weights are; other rows are not touched by them"""
    H = 96
    r = np.random.Generator(np.random.PCG64(5))
    x = r.standard_normal((4, H))
    x[1] = r.choice([-1, 1], H) * r.uniform(1e37, 3.3e38, H)
    x[3] = 0
    x[3, 40] = 3e38
    x, w = L.rounded(x, dtype), L.rounded(r.uniform(1.2, 300, H) * r.choice([-1, 1], H), "f32")
    want = L.norm(x, 1e-5, w)[0]
    want[[1, 3]] = 0
    got, _, _ = run_norm(gpu, x, dtype, dtype, w, offset=offset)
    close(got, want, L.NORM_UNITS, dtype)
    for out in ("s8", "e4m3"):
        for scaling, group in (("", 0), ("tensor", 0), ("row", 0), ("group", 32)):
            got, scale, _ = run_norm(gpu, x, dtype, out, w, scaling=scaling, group=group, given=2.0, offset=offset)
            assert (got[[1, 3]] == 0).all() and np.isfinite(got).all()
            if scaling in ("row", "group"):
                assert (scale[[1, 3]] == 0).all()
                v, s = L.quantized(want[[0, 2]], out, group)
                close(scale[[0, 2]], s, L.NORM_UNITS + 1, "f32")
                L.check_8bit(got[[0, 2]], v, 2 * L.NORM_UNITS + 4, out)


@pytest.mark.parametrize("h,weight", [(1e18, 1e21), (1e18, 1e30), (1e-30, 1e-9), (1e-38, 1e-4), (1e-20, 1e25)])
@pytest.mark.parametrize("offset", [0, 1])
def test_large_and_small_weights(gpu, h, weight, offset):
    """where the product of h and its weight is not what 32 bits hold, but the norm times the weight is"""
    H = 64
    r = np.random.Generator(np.random.PCG64(6))
    x, w = L.rounded(r.uniform(0.5, 1, (5, H)) * h, "f32"), L.rounded(r.uniform(0.5, 1, H) * weight, "f32")
    y = L.norm(x, 1e-5, w)[0]
    got, _, _ = run_norm(gpu, x, "f32", "f32", w, offset=offset)
    close(got, y, L.NORM_UNITS, "f32")
    for scaling, group in (("row", 0), ("group", 32)):
        for out in ("s8", "e4m3"):
            got, scale, _ = run_norm(gpu, x, "f32", out, w, scaling=scaling, group=group, offset=offset)
            v, s = L.quantized(y, out, group)
            if np.abs(y).max() < 1.4e-36:
                assert (scale == 0).all() and (got == 0).all()
                continue
            close(scale, s, L.NORM_UNITS + 1, "f32")
            L.check_8bit(got, v, 2 * L.NORM_UNITS + 4, out)


@pytest.mark.parametrize("scaling,group", [("row", 0), ("group", 32)])
@pytest.mark.parametrize("out", ["s8", "e4m3"])
@pytest.mark.parametrize("dtype,offset", [("f32", 0), ("f32", 1), ("bf16", 0)])
@pytest.mark.parametrize("epsilon", [1e-5, 1.0, 1e-12])
def test_small_rows_and_groups_have_scales_of_their_own(gpu, epsilon, dtype, offset, out, scaling, group):
    """Largest values from below 1.4e-36, where the scale is zero, to 1e-30, in rows whose squares vanish beside epsilon and in groups
    of ordinary rows; every row holds zeros."""
    H = 96
    most = np.concatenate([10.0 ** np.arange(-36.55, -30, 0.25), [1.3e-36, 1.36e-36, 1.44e-36, 1.6e-36, 2e-36, 2.6e-36]])  # after the norm
    r = np.random.Generator(np.random.PCG64(4))
    x = r.uniform(-1, 1, (2 * most.size, H))
    x[:, ::3] = 0
    x[:, 1::32] = np.where(r.random((2 * most.size, 3)) < 0.5, 1.0, -1.0)
    x[:most.size] *= most[:, None] * epsilon ** 0.5
    x[most.size:, 32:] *= most[:, None]  # and one group of ordinary values
    x = L.rounded(x, dtype)
    got, scale, _ = run_norm(gpu, x, dtype, out, None, scaling=scaling, group=group, offset=offset, epsilon=epsilon)
    y = L.norm(x, epsilon)[0]
    with np.errstate(all="ignore"):
        v, s = L.quantized(y, out, group)
    none = s * L.LIMIT[out] < 1.4e-36
    assert (np.abs(s * L.LIMIT[out] / 1.4e-36 - 1) > 100 * L.EPS).all()  # (none on the border)
    assert none.any() and (scale[none] == 0).all()
    close(scale[~none], s[~none], L.NORM_UNITS + 1, "f32")
    v = np.where(none.repeat(group or H, 1), 0, v)
    assert not np.isnan(got).any() and (got[v == 0] == 0).all()
    L.check_8bit(got, v, 2 * L.NORM_UNITS + 4, out)


@pytest.mark.parametrize("H", [512, 1024, 4096, 5120, 8192, 16384])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("residual", [False, True])
def test_scales_of_groups_in_rows_that_start_anywhere(gpu, H, dtype, residual):
    """every number of threads and chunks, every size of a group"""
    r = np.random.Generator(np.random.PCG64([H, residual]))
    x = L.rounded(r.standard_normal((4, H)) * np.exp(r.standard_normal((4, H // 16))).repeat(16, 1), dtype)
    res = L.rounded(r.standard_normal((4, H)), dtype) if residual else None
    w = L.rounded(r.standard_normal(H), "f32")
    y = L.norm(x, 1e-5, w, res)[0]
    for group in (16, 32, 64, 128, 256):
        for out in ("s8", "e4m3"):
            got, scale, _ = run_norm(gpu, x, dtype, out, w, residual=res, scaling="group", group=group, offset=1)
            v, s = L.quantized(y, out, group)
            close(scale, s, L.NORM_UNITS + 1, "f32")
            L.check_8bit(got, v, 2 * L.NORM_UNITS + 4, out)


def nearest_8bit(v, out):
    """`v` in 8 bits, to nearest, ties to even, saturated"""
    step = 1.0 if out == "s8" else L.step_e4m3(v)
    return np.clip(np.round(v / step) * step, -128.0 if out == "s8" else -448.0, L.LIMIT[out])


# every number of threads and chunks that a row can have
@pytest.mark.parametrize("H,groups", [(40, ()), (255, ()), (512, (16, 32, 64, 128, 256)), (1024, (16, 32, 64, 128, 256)), (2048, (32, 128, 256)),
                                      (4096, (16, 32, 64, 128, 256)), (5120, (16, 32, 64, 128, 256)), (8192, (16, 32, 64, 128, 256)),
                                      (16384, (16, 32, 64, 128, 256))])
@pytest.mark.parametrize("out", ["s8", "e4m3"])
@pytest.mark.parametrize("dtype,offset", [("bf16", 0), ("bf16", 1), ("f16", 0), ("f16", 1), ("f32", 0), ("f32", 1)])
def test_values_between_two_of_8_bits_go_to_the_even_one(gpu, H, groups, out, dtype, offset):
    """A made scale is the largest |h w| over the limit, so that the root cancels in the quotient: many quotients are ties.  h and w
    are whole numbers below 2^6 and 2^4 here: h w, of ten bits, and h w times the limit, of 17, are exact in 32 bits.  A quotient
    limit h w / m that is not a tie is at least 1 / (255 x 2^10) of itself away from one, more than 32 bits can be off: every value
    has to be the nearest one."""
    T = max(5, min(200, 80000 // H))
    r = np.random.Generator(np.random.PCG64([T, H]))
    x = np.round(r.integers(-63, 64, (T, H)) * r.random((T, 1)))
    w = r.integers(1, 16, H).astype(float)
    for group in (0,) + groups:
        got, scale, _ = run_norm(gpu, x, dtype, out, w, dtype, scaling="group" if group else "row", group=group, offset=offset)
        hw = (x * w).reshape(T, -1, group or H)
        most = np.maximum(np.abs(hw).max(2, keepdims=True), 1)
        want = nearest_8bit((hw * L.LIMIT[out] / most).reshape(T, H), out)
        bad = got != want
        assert not bad.any(), (group, bad.sum(), np.argwhere(bad)[:5], got[bad][:5], want[bad][:5])
        close(scale, np.abs(L.norm(x, 1e-5, w)[0]).reshape(T, -1, group or H).max(2) / L.LIMIT[out], L.NORM_UNITS + 1, "f32")


@pytest.mark.parametrize("dtype,offset", [("f32", 0), ("bf16", 0), ("bf16", 1)])
@pytest.mark.parametrize("T,H", [(5, 96), (700, 40)])
def test_gradient_of_rows_whose_squares_exceed_32_bits(gpu, T, H, dtype, offset):
    """zeros besides what comes along the residual path, and nothing in the weights' gradient"""
    r = np.random.Generator(np.random.PCG64(7))
    h, dy, dsum = r.standard_normal((T, H)), r.standard_normal((T, H)) * 3, r.standard_normal((T, H))
    over = np.arange(T) % 4 == 1
    h[over] = r.choice([-1, 1], (over.sum(), H)) * r.uniform(1e37, 3.3e38, (over.sum(), H))
    h, dy, dsum = (L.rounded(v, dtype) for v in (h, dy, dsum))
    w = L.rounded(r.uniform(1.2, 300, H), "f32")
    for add in (None, dsum):
        got, gotw = run_backward(gpu, h, dy, dtype, w, "f32", add, "f32", offset=offset)
        assert np.array_equal(got[over], np.zeros_like(got[over]) if add is None else dsum[over])
        check_backward(got[~over], gotw, h[~over], dy[~over], dtype, w, None if add is None else dsum[~over], "f32")


@pytest.mark.parametrize("H,offset", [(96, 0), (96, 1), (2048, 0)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_infinities_and_nan_stay_where_they_are(gpu, H, offset, dtype):
    """rows with an infinity are zeros but for a NaN where it is, those with a NaN are NaN; an infinite value makes an infinite scale"""
    r = np.random.Generator(np.random.PCG64(8))
    x, w = L.rounded(r.standard_normal((5, H)), dtype), L.rounded(r.standard_normal(H), "f32")
    x[1, 7], x[2, 40], x[3, 50] = np.inf, -np.inf, np.nan
    want = L.norm(x[[0, 4]], 1e-5, w)[0]
    got, _, _ = run_norm(gpu, x, dtype, dtype, w, offset=offset)
    close(got[[0, 4]], want, L.NORM_UNITS, dtype)
    at = np.isnan(got)
    assert at[3].all() and at[1].sum() == at[2].sum() == 1 and at[1, 7] and at[2, 40] and (got[1:3][~at[1:3]] == 0).all()
    got, scale, _ = run_norm(gpu, x, dtype, "e4m3", w, scaling="group", group=32, offset=offset)
    of = np.arange(H) // 32
    assert np.array_equal(np.isnan(got[1]), of == 0) and np.array_equal(np.isnan(got[2]), of == 1) and np.isnan(got[3]).all()
    assert np.array_equal(np.isnan(scale[1]), np.arange(H // 32) == 0) and (scale[1, 1:] == 0).all() and np.isnan(scale[3]).all()
    # the gradient: the same, besides what comes along the residual path
    dy, dsum = (L.rounded(r.standard_normal((5, H)), dtype) for _ in range(2))
    got, gotw = run_backward(gpu, x, dy, dtype, w, "f32", dsum, "f32", offset=offset)
    at = np.isnan(got)
    assert at[3].all() and at[1].sum() == at[2].sum() == 1 and at[1, 7] and at[2, 40] and np.array_equal(got[1:3][~at[1:3]], dsum[1:3][~at[1:3]])
    # a weight that takes the value beyond 32 bits
    x, w = np.where(np.isfinite(x), x, 0), w.copy()
    x[0, 3], w[3] = 100.0, 3.4e38
    w = L.rounded(w, "f32")
    for out in ("s8", "e4m3"):
        got, scale, _ = run_norm(gpu, x, dtype, out, w, scaling="group", group=32, offset=offset)
        assert scale[0, 0] == np.inf and np.isfinite(scale[0, 1:]).all()
        assert np.isnan(got[0, :32]).all() if out == "e4m3" else (got[0, :32] == 0).all()
        assert np.isfinite(got[0, 32:]).all()

"""Low-rank adapters on a device: the base beside products of any size, rows beside other rows."""
import numpy as np
import pytest

import layer_ref as L
from test_low_rank_gpu import make, run, verify

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,r", [(40, 8), (40, 64), (1200, 16), (600, 128)])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("offset", [0, 1])
def test_a_large_base_beside_small_products(gpu, T, r, dtype, offset):
    """products down to 2^-70 of the base's 32-bit values, and the other way round"""
    n, K, N = 3, 64, 72
    x, index, down, up, scale, g = make(T, n, K, r, N, dtype)
    x = L.rounded(x * 10.0 ** g.uniform(-7, 1, (T, 1)), dtype)
    down, up = L.rounded(down * 1e-2, dtype), L.rounded(up * 1e-1, dtype)
    scale = L.rounded(scale * 10.0 ** -g.integers(0, 4, n), "f32")
    base = L.rounded(g.standard_normal((T, N)) * 10.0 ** g.uniform(-37, 37, (T, 1)), "f32")
    got = run(gpu, x, index, down, up, dtype, "f32", scale, base, "middle", "middle", offset, offset)
    assert np.isfinite(got).all()
    verify(got, x, index, down, up, scale, base, dtype, "f32")


@pytest.mark.parametrize("T,r", [(40, 8), (600, 128)])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_small_products_keep_their_bits(gpu, T, r, dtype):
    """the first product times an adapter's scale down to 1e-30: in 32-bit results as exact as any other"""
    x, index, down, up, scale, g = make(T, 8, 64, r, 72, dtype)
    scale = L.rounded(scale * 10.0 ** -g.uniform(10, 30, 8), "f32")
    got = run(gpu, x, index, down, up, dtype, "f32", scale, None, "middle", "middle")
    verify(got, x, index, down, up, scale, None, dtype, "f32")


@pytest.mark.parametrize("T,r,out", [(300, 16, "f32"), (300, 128, "bf16"), (1100, 16, "bf16"), (1500, 32, "f32"), (700, 64, "bf16")])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_a_row_does_not_depend_on_its_neighbours(gpu, T, r, out, dtype):
    """the same bits where the rows stand in another order, and where all but some are replaced, in one launch and in two"""
    out = dtype if out == "bf16" else out
    x, index, down, up, scale, g = make(T, 6, 512, r, 264, dtype)
    base = L.rounded(g.standard_normal((T, 264)), out)
    first = run(gpu, x, index, down, up, dtype, out, scale, base)
    verify(first, x, index, down, up, scale, base, dtype, out)
    order = g.permutation(T)
    assert np.array_equal(run(gpu, x[order], index[order], down, up, dtype, out, scale, base[order]), first[order])
    kept = g.random(T) < 0.3
    other, others = x.copy(), index.copy()
    other[~kept] = L.rounded(g.standard_normal((T, 512)), dtype)[~kept]
    other[np.argmin(kept)] = np.nan
    others[~kept] = g.integers(-1, 6, T)[~kept]
    assert np.array_equal(run(gpu, other, others, down, up, dtype, out, scale, base)[kept], first[kept])


@pytest.mark.parametrize("T", [200, 1100])
@pytest.mark.parametrize("in_place", [False, True])
def test_indices_that_name_no_adapter(gpu, T, in_place):
    n = 4
    x, index, down, up, scale, g = make(T, n, 128, 16, 264, "bf16", none=0)
    none = [n, -1, 1 << 30, -(1 << 31), n + 1, 99, -2, (1 << 31) - 1, 1024, 65536]
    for i, value in enumerate(none):
        index[i::17] = value
    base = L.rounded(g.standard_normal((T, 264)), "bf16")
    got = run(gpu, x, index, down, up, "bf16", "bf16", scale, base, in_place=in_place)
    verify(got, x, index, down, up, scale, base, "bf16", "bf16")
    off = (index < 0) | (index >= n)
    assert off.mean() > 0.5 and np.array_equal(got[off], base[off])

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

"""The router with a bias on the choice and groups of experts: what needs no device - the plain form, descriptors, refusals."""
import ctypes as C
import os
import re

import numpy as np
import pytest

import layer_ref as L
import token_ref as R
from test_dependent_launch import NON_COHERENT, _functions, _reachable, _source

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F32, BF16, S32 = 3, 2, 4


def test_plain_form():
    x = np.array([[3.0, 0, 0, 2.9, 2.9, 2.9, 1, 1], [1, 1, 1, 1, 1, 1, 1, 1], [-np.inf] * 6 + [0, np.nan]])
    assert L.choose(x, None, "softmax", 3).tolist() == [[0, 3, 4], [0, 1, 2], [6, -1, -1]]
    assert L.choose(x, None, "sigmoid", 2, 4, 1, 1).tolist() == [[0, 1], [0, 1], [6, -1]]  # groups of two: 3.0 leads
    assert L.choose(x, None, "sigmoid", 2, 4, 1, 2).tolist() == [[4, 5], [0, 1], [6, -1]]  # two of 2.9 lead
    bias = np.array([0, 0, 0, 0, 0, 0, 1.0, -np.inf])
    assert L.choose(x, bias, "sigmoid", 3).tolist() == [[6, 0, 3], [6, 0, 1], [6, -1, -1]]
    # without a bias and groups it is the plain router
    r = np.random.Generator(np.random.PCG64(1))
    x = r.standard_normal((50, 40))
    assert np.array_equal(L.choose(x, None, "softmax", 7), R.choose(x, 7))
    assert np.array_equal(L.choose(x, np.full(40, 0.25), "sigmoid", 7, 5, 5, 2), R.choose(x, 7))


def test_descriptors_and_refusals(host_engine):
    from onednn_b200 import api
    md, O = api.memory.desc, api.RUNTIME_DIM_VAL
    ok, bad, no = api.success, api.invalid_arguments, api.unimplemented

    def make(T=5, E=16, k=4, bias=None, **kw):
        try:
            api.moe_route.primitive_desc(host_engine, md((T, E), F32, (E, 1)), md((T, k), F32, (k, 1)), md((T, k), S32, (k, 1)),
                                         bias_md=bias, **kw)
        except api.error as e:
            return e.status
        return ok

    def groups(n, kept, best=1):
        return dict(groups=n, groups_kept=kept, group_best=best)

    b = md((16,), F32, (1,))
    for want, kw in [
            (ok, dict(bias=b)), (bad, dict(bias=md((15,), F32, (1,)))), (no, dict(bias=md((16,), BF16, (1,)))),
            (no, dict(bias=md((16,), F32, (2,)))), (bad, dict(bias=md((1, 16), F32, (16, 1)))),
            (ok, groups(4, 2, 2)), (ok, dict(bias=b, **groups(4, 4, 1))), (bad, groups(4, 5)), (bad, groups(4, 0)), (bad, groups(0, 0)),
            (bad, groups(-1, 1)), (bad, groups(5, 2)), (bad, groups(4, 2, 0)), (bad, groups(4, 2, 3)), (bad, dict(k=9, **groups(4, 2))),
            (ok, dict(k=8, **groups(4, 2))), (ok, groups(16, 4, 2)), (ok, dict(E=128, **groups(32, 4))), (no, dict(E=128, **groups(64, 4))),
            (ok, dict(T=0, bias=b)), (bad, dict(k=17, bias=b)), (bad, dict(scale=float("inf"), bias=b)), (bad, dict(scoring=2, bias=b))]:
        assert make(**kw) == want, kw
    pd = api.moe_route.primitive_desc(host_engine, md((O, O), F32, (O, 1)), md((O, 4), F32, (4, 1)), md((O, 4), S32, (4, 1)),
                                      bias_md=md((O,), F32, (1,)), groups=4, groups_kept=2)
    assert pd.query_md(255, api.ARG_BIAS).get_dims() == (O,) and pd.impl_info_str() == "cuda:simt:moe_route"
    h, f = C.c_void_p(), api.lib().dnnl_cuda_interop_moe_route_v2_primitive_desc_create
    m, w, i = md((5, 16), F32, (16, 1)), md((5, 4), F32, (4, 1)), md((5, 4), S32, (4, 1))
    assert f(C.byref(h), host_engine._h, m._h, None, w._h, None, 0, 1, 1.0, 4, 2, 2, None) == bad
    assert f(C.byref(h), host_engine._h, None, None, w._h, i._h, 0, 1, 1.0, 4, 2, 2, None) == bad


@pytest.mark.parametrize("file", ["moe_route_groups.cu", "moe_route.cu"])
def test_kernels_read_with_coherent_loads(file):
    kernels = _reachable(file)
    assert kernels
    for name, text in kernels.items():
        assert not NON_COHERENT.findall(text), name


@pytest.mark.parametrize("file", ["moe_route_groups.cu", "route_keys.cuh"])
def test_every_function_is_called(file):
    sources = os.path.join(ROOT, "onednn_b200", "csrc")
    text = "".join(_source(f) for f in os.listdir(sources) if f.endswith((".cu", ".cuh", ".h", ".hpp")))
    assert not [n for n in _functions(_source(file)) if len(re.findall(r"\b%s\b" % n, text)) < 2]

"""Low-rank adapters: what needs no device - the plain form, descriptors, refusals, queries, and how the kernel reads what the
call before it wrote."""
import ctypes as C
import os
import re

import numpy as np

import layer_ref as L
from test_dependent_launch import NON_COHERENT, _functions, _reachable, _source

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F16, BF16, F32, S32, S8 = 1, 2, 3, 4, 5


def test_plain_form_and_its_gradient_against_differences():
    r = np.random.Generator(np.random.PCG64(2))
    T, n, K, N, k = 7, 3, 5, 6, 2
    x, down, up = r.standard_normal((T, K)), r.standard_normal((n, K, k)), r.standard_normal((n, k, N))
    scale, base, g = r.random(n) + 0.5, r.standard_normal((T, N)), r.standard_normal((T, N))
    index = np.array([0, 2, -1, 2, 1, 3, 0])
    y, _, _ = L.low_rank(x, index, down, up, scale, base)
    for t in range(T):
        i = index[t]
        want = base[t] + (scale[i] * (x[t] @ down[i] @ up[i]) if 0 <= i < n else 0)
        assert np.allclose(y[t], want, rtol=1e-13)
    # the gradient of x is the same operator with the factors transposed and exchanged
    dx, _, _ = L.low_rank(g, index, up.transpose(0, 2, 1), down.transpose(0, 2, 1), scale)
    step = 1e-6
    for t in range(T):
        for c in range(K):
            p, m = x.copy(), x.copy()
            p[t, c] += step
            m[t, c] -= step
            num = ((L.low_rank(p, index, down, up, scale)[0] - L.low_rank(m, index, down, up, scale)[0]) * g).sum() / (2 * step)
            assert abs(num - dx[t, c]) < 1e-7


def test_descriptors_and_refusals(host_engine):
    from onednn_b200 import api
    md, O = api.memory.desc, api.RUNTIME_DIM_VAL
    ok, bad, no = api.success, api.invalid_arguments, api.unimplemented

    def make(T=5, K=32, n=3, r=8, N=48, dt=BF16, out=BF16, idx=None, down=None, up=None, dst=None, base=None, src=None, attr=None):
        try:
            return api.success, api.low_rank_adapter.primitive_desc(
                host_engine, src or md((T, K), dt, (K, 1)), idx or md((T,), S32, (1,)), down or md((n, K, r), dt, (K * r, r, 1)),
                up or md((n, r, N), dt, (r * N, N, 1)), dst or md((T, N), out, (N, 1)), base_md=base, attr=attr)
        except api.error as e:
            return e.status, None

    for want, kw in [
            (ok, {}), (ok, dict(dt=F16, out=F16)), (ok, dict(out=F32)), (no, dict(out=F16)), (no, dict(dt=F32, out=F32)), (no, dict(dt=S8, out=F32)),
            (ok, dict(r=128)), (no, dict(r=129)), (ok, dict(n=1)), (ok, dict(T=0)), (ok, dict(K=1, N=1, r=1)),
            (bad, dict(idx=md((4,), S32, (1,)))), (no, dict(idx=md((5,), F32, (1,)))), (bad, dict(idx=md((5, 1), S32, (1, 1)))),
            (no, dict(idx=md((5,), S32, (2,)))), (bad, dict(down=md((3, 31, 8), BF16, (248, 8, 1)))), (bad, dict(down=md((2, 32, 8), BF16, (256, 8, 1)))),
            (bad, dict(up=md((3, 9, 48), BF16, (432, 48, 1)))), (bad, dict(up=md((3, 8, 47), BF16, (400, 48, 1)))),
            (ok, dict(down=md((3, 32, 8), BF16, (256, 1, 32)))), (ok, dict(down=md((3, 32, 8), BF16, (1, 3, 96)))), (no, dict(down=md((3, 32, 8), F16, (256, 8, 1)))),
            (bad, dict(down=md((3, 256), BF16, (256, 1)))), (ok, dict(dst=md((5, 48), BF16, (50, 1)))), (no, dict(dst=md((5, 48), BF16, (1, 5)))),
            (no, dict(dst=md((5, 48), BF16, (0, 1)))), (ok, dict(src=md((5, 32), BF16, (0, 1)))), (bad, dict(src=md((6, 32), BF16, (32, 1)))),
            (ok, dict(base=md((5, 48), BF16, (48, 1)))), (no, dict(base=md((5, 48), F32, (48, 1)))), (bad, dict(base=md((5, 40), BF16, (48, 1))))]:
        assert make(**kw)[0] == want, kw
    # open rows, and an adapter's scale
    attr = api.primitive_attr()
    attr.set_scales(api.ARG_WEIGHTS, 1)
    st, pd = make(src=md((O, 32), BF16, (O, 1)), idx=md((O,), S32, (1,)), dst=md((O, 48), BF16, (O, 1)), attr=attr)
    scales = api.ARG_ATTR_SCALES | api.ARG_WEIGHTS
    assert st == ok and pd.query_md(255, scales) == md((3, 1, 1), F32, (1, 1, 1)) and pd.impl_info_str() == "cuda:simt:low_rank_adapter"
    assert pd.query_md(131, 1) == md((3, 8, 48), BF16, (384, 48, 1)) and pd.query_md(131, 0) == md((3, 32, 8), BF16, (256, 8, 1))
    assert [api.lib().dnnl_primitive_desc_query_s32(pd._h, q, 0) for q in (3, 4)] == [5, 1]
    for set_ in (lambda a: a.set_scales(api.ARG_WEIGHTS, 0), lambda a: a.set_scales(api.ARG_WEIGHTS, 1, (), BF16), lambda a: a.set_scales(api.ARG_DST, 0),
                 lambda a: a.set_scales(api.ARG_WEIGHTS, 6, (8, 8)), lambda a: a.set_scales(api.ARG_WEIGHTS, 1, qmode=api.quantization_mode.dynamic_fp),
                 lambda a: a.set_fpmath_mode(api.fpmath_mode.bf16, True)):
        attr = api.primitive_attr()
        set_(attr)
        assert make(attr=attr)[0] == no
    h, f = C.c_void_p(), api.lib().dnnl_cuda_interop_low_rank_adapter_primitive_desc_create
    m = md((5, 32), BF16, (32, 1))
    assert f(C.byref(h), host_engine._h, m._h, None, m._h, m._h, None, m._h, None) == bad
    api.lib().dnnl_prim_kind2str.restype = C.c_char_p
    assert api.lib().dnnl_prim_kind2str(0x10012) == b"low_rank_adapter"


def test_kernels_read_with_coherent_loads():
    kernels = _reachable("low_rank.cu")
    assert set(kernels) == {"low_rank_few_kernel", "low_rank_down_kernel", "low_rank_up_kernel"}
    for name, text in kernels.items():
        assert not NON_COHERENT.findall(text), name


def test_every_function_is_called():
    sources = os.path.join(ROOT, "onednn_b200", "csrc")
    text = "".join(_source(f) for f in os.listdir(sources) if f.endswith((".cu", ".cuh", ".h", ".hpp")))
    assert not [n for n in _functions(_source("low_rank.cu")) if len(re.findall(r"\b%s\b" % n, text)) < 2]


def test_cluster_barriers_come_in_pairs():
    """each arrival at the cluster's barrier has its wait: one right behind it, one before the sums are overwritten or the CTA ends"""
    body = _functions(_source("low_rank.cu"))["low_rank_few_kernel"]
    assert len(re.findall(r"cluster_arrive\(\)", body)) == 2
    assert re.search(r"if \(arrived\) cluster_wait\(\);.*cluster_arrive\(\);\s*cluster_wait\(\);.*cluster_arrive\(\);\s*arrived = true;", body, re.S)
    assert re.search(r"if \(arrived\) cluster_wait\(\);\s*\}?\s*$", body)

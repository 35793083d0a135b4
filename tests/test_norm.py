"""The root-mean-square norm and its gradient: what needs no device - the plain forms that the device is compared with,
descriptors, refusals, queries, and how the kernels read what the call before them wrote."""
import ctypes as C
import os
import re
import shutil
import subprocess

import numpy as np
import pytest

import layer_ref as L
from test_dependent_launch import NON_COHERENT, _functions, _reachable, _source

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F16, BF16, F32, S32, S8, U8, E5M2, E4M3 = 1, 2, 3, 4, 5, 6, 9, 10


def test_gradient_formula_against_differences():
    r = np.random.Generator(np.random.PCG64(3))
    T, H, step = 4, 9, 1e-6
    h, dy, w, dsum = (r.standard_normal(s) for s in ((T, H), (T, H), (H,), (T, H)))
    h[2] *= 1e-3
    dh, dw, _, _ = L.norm_backward(h, dy, 1e-5, w, dsum)

    def value(h, w):
        return (L.norm(h, 1e-5, w)[0] * dy).sum() + (h * dsum).sum()

    for t in range(T):
        for i in range(H):
            at = [h.copy(), h.copy()]
            at[0][t, i] += step * (1 if t != 2 else 1e-3)
            at[1][t, i] -= step * (1 if t != 2 else 1e-3)
            num = (value(at[0], w) - value(at[1], w)) / (at[0][t, i] - at[1][t, i])
            assert abs(num - dh[t, i]) < 1e-6 * max(1, abs(dh).max()), (t, i)
    for i in range(H):
        at = [w.copy(), w.copy()]
        at[0][i] += step
        at[1][i] -= step
        assert abs((value(h, at[0]) - value(h, at[1])) / (2 * step) - dw[i]) < 1e-7


def test_check_8bit_knows_a_wrong_value():
    v = np.array([[0.49, 1.5, -2.4, 300.0, 1e-9]])
    L.check_8bit(np.array([[0, 2, -2, 127, 0]]), v, 40, "s8")
    L.check_8bit(np.array([[0.5, 1.5, -2.5, 288.0, 0]]), v, 40, "e4m3")
    for q in ([[1, 2, -2, 127, 0]], [[0, 2, -2, 126, 0]], [[0, 1, -3, 127, 0]]):
        with pytest.raises(AssertionError):
            L.check_8bit(np.array(q, float), v, 40, "s8")


def make(api, eng, src=(5, 64), dst=None, dt=BF16, out=BF16, eps=1e-5, src_stride=None, dst_stride=None, weights=None,
         residual=None, total=None, scales=None):
    md = api.memory.desc
    attr = None
    if scales is not None:
        attr = api.primitive_attr()
        attr.set_scales(api.ARG_DST, *scales[0], **scales[1])
    dst = src if dst is None else dst
    return api.rms_norm.primitive_desc(
        eng, md(src, dt, src_stride or (src[1], 1)), md(dst, out, dst_stride or (dst[1], 1)), eps, weights_md=weights,
        residual_md=residual, sum_md=total, attr=attr)


def status(api, f):
    try:
        f()
    except api.error as e:
        return e.status
    return api.success


def test_descriptors_and_refusals(host_engine):
    from onednn_b200 import api
    md, O, eng = api.memory.desc, api.RUNTIME_DIM_VAL, host_engine
    mode = api.quantization_mode
    dynamic = dict(qmode=mode.dynamic_fp)
    ok, bad, no = api.success, api.invalid_arguments, api.unimplemented
    for want, kw in [
            (ok, {}), (ok, dict(dt=F32, out=F32)), (ok, dict(out=F32)), (ok, dict(out=S8)), (ok, dict(out=E4M3)),
            (no, dict(out=F16)), (no, dict(out=U8)), (no, dict(out=E5M2)), (no, dict(dt=S8, out=S8)), (no, dict(dt=F32, out=BF16)),
            (bad, dict(dst=(4, 64))), (bad, dict(dst=(5, 63))), (bad, dict(eps=0.0)), (bad, dict(eps=-1.0)),
            (bad, dict(eps=float("nan"))), (bad, dict(eps=float("inf"))), (bad, dict(eps=1e-60)),
            (ok, dict(src=(0, 64))), (bad, dict(src=(5, 0))), (ok, dict(src=(1, 16384))), (no, dict(src=(1, 16385))),
            (no, dict(src_stride=(1, 5))), (no, dict(dst_stride=(0, 1))), (ok, dict(src_stride=(0, 1))),
            (ok, dict(weights=md((64,), BF16, (1,)))), (ok, dict(weights=md((64,), F32, (1,)))),
            (no, dict(weights=md((64,), F16, (1,)))), (bad, dict(weights=md((63,), F32, (1,)))),
            (bad, dict(weights=md((1, 64), F32, (64, 1)))), (no, dict(weights=md((64,), F32, (2,)))),
            (ok, dict(residual=md((5, 64), BF16, (70, 1)))), (no, dict(residual=md((5, 64), F32, (64, 1)))),
            (bad, dict(residual=md((5, 60), BF16, (64, 1)))), (ok, dict(total=md((5, 64), BF16, (70, 1)))),
            (no, dict(total=md((5, 64), F32, (64, 1)))), (no, dict(total=md((5, 64), BF16, (0, 1)))),
            (ok, dict(out=S8, scales=((0,), {}))), (ok, dict(out=E4M3, scales=((1,), dynamic))),
            (ok, dict(out=S8, scales=((3, (1, 16)), dynamic))), (no, dict(out=S8, scales=((3, (1, 8)), dynamic))),
            (no, dict(out=S8, scales=((3, (1, 48)), dynamic))), (bad, dict(out=S8, scales=((3, (1, 128)), dynamic))),
            (no, dict(out=S8, scales=((3, (2, 16)), dynamic))), (no, dict(out=S8, scales=((3,), dynamic))),
            (no, dict(out=S8, scales=((1,), {}))), (no, dict(out=S8, scales=((0,), dynamic))),
            (no, dict(out=S8, scales=((1,), dict(qmode=mode.dynamic_mx)))), (no, dict(out=S8, scales=((2,), dynamic))),
            (no, dict(out=BF16, scales=((0,), {}))), (no, dict(out=S8, scales=((0, (), BF16), {}))),
            (no, dict(out=S8, scales=((0,), dict(is_on_host=True)))),
            (ok, dict(src=(O, 64), src_stride=(O, 1), dst_stride=(O, 1))),
            (ok, dict(src=(O, O), src_stride=(O, 1), dst_stride=(O, 1), out=S8, scales=((3, (1, 128)), dynamic)))]:
        assert status(api, lambda: make(api, eng, **kw)) == want, kw
    m = md((5, 64), BF16, (64, 1))
    w = md((64,), F32, (1,))

    def back(ddst=m, src=m, dsrc=m, eps=1e-5, **kw):
        return status(api, lambda: api.rms_norm_backward.primitive_desc(eng, ddst, src, dsrc, eps, **kw))

    assert back() == ok and back(weights_md=w, diff_weights_md=w, diff_sum_md=m) == ok
    assert back(diff_weights_md=md((64,), BF16, (1,))) == ok and back(diff_weights_md=md((64,), F16, (1,))) == no
    assert back(eps=0.0) == bad and back(ddst=md((5, 63), BF16, (64, 1))) == bad and back(src=md((5, 64), F32, (64, 1))) == no
    assert back(dsrc=md((5, 64), BF16, (0, 1))) == no and back(diff_weights_md=md((63,), F32, (1,))) == bad
    open_rows = md((O, 64), BF16, (O, 1))
    assert back(open_rows, open_rows, open_rows, diff_weights_md=w) == ok
    open_all, open_w = md((O, O), BF16, (O, 1)), md((O,), F32, (1,))
    assert back(open_all, open_all, open_all) == ok and back(open_all, open_all, open_all, diff_weights_md=open_w) == no
    # attributes: the scales of dst and the scratchpad mode, nothing else
    for arg in (api.ARG_SRC, api.ARG_WEIGHTS):
        attr = api.primitive_attr()
        attr.set_scales(arg, 0)
        assert status(api, lambda: api.rms_norm.primitive_desc(eng, m, md((5, 64), S8, (64, 1)), 1e-5, attr=attr)) == no
    attr = api.primitive_attr()
    attr.set_scales(api.ARG_DST, 0)
    assert back(attr=attr) == no
    attr = api.primitive_attr()
    attr.set_fpmath_mode(api.fpmath_mode.bf16, False)
    assert status(api, lambda: api.rms_norm.primitive_desc(eng, m, m, 1e-5, attr=attr)) == no
    # C callers' null pointers
    h, f = C.c_void_p(), api.lib().dnnl_cuda_interop_rms_norm_primitive_desc_create
    assert f(None, eng._h, m._h, None, None, m._h, None, 1e-5, None) == bad
    assert f(C.byref(h), None, m._h, None, None, m._h, None, 1e-5, None) == bad
    assert f(C.byref(h), eng._h, None, None, None, m._h, None, 1e-5, None) == bad
    assert f(C.byref(h), eng._h, m._h, None, None, None, None, 1e-5, None) == bad


def test_queries(host_engine):
    from onednn_b200 import api
    md, eng, O = api.memory.desc, host_engine, api.RUNTIME_DIM_VAL
    dynamic = dict(qmode=api.quantization_mode.dynamic_fp)
    m, w = md((6, 256), BF16, (256, 1)), md((256,), F32, (1,))
    pd = make(api, eng, src=(6, 256), out=S8, weights=w, residual=m, total=m, scales=((3, (1, 64)), dynamic))
    scales = api.ARG_ATTR_SCALES | api.ARG_DST
    assert pd.query_md(255, scales) == md((6, 4), F32, (4, 1)) and pd.query_md(255, api.ARG_SRC_2) == m
    assert pd.impl_info_str() == "cuda:simt:rms_norm"
    value = C.c_int()
    lib = api.lib()
    assert lib.dnnl_primitive_desc_query(pd._h, 2, 0, C.byref(value)) == 0 and value.value == 0x10010
    counts = [lib.dnnl_primitive_desc_query_s32(pd._h, q, 0) for q in (3, 4)]
    assert counts == [3, 3]  # src, residual, weights; dst, its scales, the sum
    pd = make(api, eng, src=(6, 256), out=S8, scales=((1,), dynamic))
    assert pd.query_md(255, scales) == md((6, 1), F32, (1, 1))
    pd = make(api, eng, src=(6, 256), out=S8, scales=((0,), {}))
    assert pd.query_md(255, scales) == md((1, 1), F32, (1, 1))
    assert [lib.dnnl_primitive_desc_query_s32(pd._h, q, 0) for q in (3, 4)] == [2, 1]
    pd = make(api, eng, src=(O, 256), src_stride=(O, 1), dst_stride=(O, 1), out=S8, scales=((1,), dynamic))
    assert pd.query_md(255, scales).get_dims() == (O, 1)
    lib.dnnl_prim_kind2str.restype = C.c_char_p
    assert [lib.dnnl_prim_kind2str(k) for k in (0x1000f, 0x10010, 0x10011)] == [b"unknown prim_kind", b"rms_norm", b"rms_norm_backward"]
    # the gradient's scratchpad: one part of the weights' gradient for each CTA
    attr = api.primitive_attr()
    attr.set_scratchpad_mode(api.SCRATCHPAD_MODE_USER)
    back = api.rms_norm_backward.primitive_desc
    assert back(eng, m, m, m, 1e-5, diff_weights_md=w, attr=attr).query_md(255, api.ARG_SCRATCHPAD).get_dims()[0] % (256 * 4) == 0
    assert back(eng, m, m, m, 1e-5, attr=attr).query_md(255, api.ARG_SCRATCHPAD).get_ndims() == 0


def test_kernels_read_with_coherent_loads():
    kernels = _reachable("rms_norm.cu")
    assert set(kernels) == {"rms_norm_kernel", "rms_norm_backward_kernel", "rms_norm_weights_kernel"}
    for name, text in kernels.items():
        assert not NON_COHERENT.findall(text), name


def test_every_function_is_called():
    sources = os.path.join(ROOT, "onednn_b200", "csrc")
    text = "".join(_source(f) for f in os.listdir(sources) if f.endswith((".cu", ".cuh", ".h", ".hpp")))
    assert not [n for n in _functions(_source("rms_norm.cu")) if len(re.findall(r"\b%s\b" % n, text)) < 2]


def test_the_header_compiles_as_c(tmp_path):
    (tmp_path / "h.c").write_text('#include "dnnl_b200.h"\nint main(void) { return dnnl_cuda_interop_rms_norm != 0x10010; }\n')
    exe = str(tmp_path / "h")
    r = subprocess.run([shutil.which("gcc") or "/usr/bin/gcc", "-std=c99", str(tmp_path / "h.c"), "-I" + os.path.join(ROOT, "include"),
                        "-o", exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-2000:]
    assert subprocess.run([exe], timeout=60).returncode == 0

"""The operators around an expert layer's products, and dropout: what needs no device - the plain forms the device is
compared with, descriptors, refusals, queries, and how the kernels read what the call before them wrote."""
import ctypes as C

import numpy as np
import pytest

import token_ref as R
from test_dependent_launch import NON_COHERENT, _reachable


def test_philox_known_answers():
    """the published vectors of Philox4x32-10: all zero, all ones, and digits of pi"""
    assert [int(w) for w in R.philox_words(0, 0, 0, 4)] == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]
    ones = (1 << 64) - 1  # (counter words 0 and 1 are the block's number)
    assert [int(w) for w in R.philox_blocks(ones, ones, np.array([ones], np.uint64))[0]] == [
        0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]
    assert [int(w) for w in R.philox_blocks(0x299f31d0a4093822, 0x0370734413198a2e, np.array([0x85a308d3243f6a88], np.uint64))[0]] == [
        0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1]
    assert np.array_equal(R.philox_words(5, 6, 0, 40)[7:22], R.philox_words(5, 6, 7, 15))


@pytest.mark.parametrize("scoring,normalize", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
def test_route_gradient_formula_against_differences(scoring, normalize):
    r = np.random.Generator(np.random.PCG64(4))
    T, E, k, h = 5, 17, 4, 1e-5
    x, g = r.standard_normal((T, E)), r.standard_normal((T, k))
    x[2, 3:9] = -np.inf
    idx = R.choose(x, k)
    idx[3, 2:] = -1
    d, _ = R.route_backward(x, idx, g, scoring, normalize, 1.5)
    num = np.zeros((T, E))
    for t in range(T):
        for e in range(E):
            f = []
            for s in (h, -h):
                y = x.copy()
                y[t, e] += s
                f.append((R.route_weights(y, idx, scoring, normalize, 1.5) * g).sum())
            num[t, e] = (f[0] - f[1]) / (2 * h)
    assert np.abs(d - num).max() < 1e-8


def test_sort_of_slots():
    ends, pos, order = R.sort_slots(np.array([[1, 0], [1, -1], [5, 0]]), 3)
    assert ends.tolist() == [2, 4, 4] and pos.tolist() == [[2, 0], [3, -1], [-1, 1]] and order.tolist() == [1, 5, 0, 2]


# ------------------------------------------------------------------------------------- descriptors and refusals

F16, BF16, F32, S32, S8, S64 = 1, 2, 3, 4, 5, 16


def mats(api):
    md = api.memory.desc

    def m(rows, cols, dt=F32, pitch=None, inner=1):
        return md((rows, cols), dt, (cols if pitch is None else pitch, inner))
    return md, m


def route(api, eng, logits, weights, indices, **kw):
    return api.moe_route.primitive_desc(eng, logits, weights, indices, **kw)


def test_descriptors_can_be_queried(host_engine):
    from onednn_b200 import api
    md, m = mats(api)
    eng = host_engine
    pd = route(api, eng, m(5, 8, BF16), m(5, 2), m(5, 2, S32))
    assert pd.impl_info_str() == "cuda:simt:moe_route" and not pd.next_impl()
    assert pd.src_desc() == m(5, 8, BF16) and pd.dst_desc() == m(5, 2)
    assert pd.query_md(255, api.ARG_DST_1) == m(5, 2, S32) and pd.weights_desc() is None
    g = md.grouped((10, 4), BF16, 0, 8)
    pd = api.moe_combine.primitive_desc(eng, g, m(5, 2, S32), m(5, 4, BF16), weights_md=m(5, 2), residual_md=m(5, 4, BF16), dropout_p=0.1)
    assert pd.weights_desc() == m(5, 2) and pd.query_md(129, 2) == m(5, 4, BF16)
    assert pd.query_md(255, api.ARG_ATTR_DROPOUT_SEED) == md((2,), S64, (1,))
    lib = api.lib()
    assert lib.dnnl_primitive_desc_query_s32(pd._h, 3, 0) == 5 and lib.dnnl_primitive_desc_query_s32(pd._h, 4, 0) == 1
    kind = C.c_int()
    assert lib.dnnl_primitive_desc_query(pd._h, 2, 0, C.byref(kind)) == 0
    lib.dnnl_prim_kind2str.restype = C.c_char_p
    assert lib.dnnl_prim_kind2str(kind) == b"moe_combine"
    assert api.moe_combine.primitive_desc(eng, g, m(5, 2, S32), m(5, 4)).query_md(255, api.ARG_ATTR_DROPOUT_SEED).get_ndims() == 0
    pd = api.moe_combine_backward.primitive_desc(eng, m(5, 4), g, m(5, 2, S32), m(5, 2), g, m(5, 2), dropout_p=0.5)
    assert pd.query_md(134) == m(5, 4) and pd.query_md(132) == m(5, 2) and pd.query_md(130) == g
    api.dropout.primitive_desc(eng, m(3, 7, F16, 9), m(3, 7, F16), 0.0)
    api.moe_dispatch.primitive_desc(eng, m(5, 4, S8, 0), m(5, 2, S32), md.grouped((10, 4), S8, 0, 8), m(5, 2, S32))


def test_refusals(host_engine):
    from onednn_b200 import api
    md, m = mats(api)
    eng, bad, nb = host_engine, api.invalid_arguments, api.unimplemented
    O = api.RUNTIME_DIM_VAL

    def refuse(status, f):
        with pytest.raises(api.error) as e:
            f()
        assert e.value.status == status

    w, i = m(5, 2), m(5, 2, S32)
    for status, args, kw in (
            (bad, (m(6, 8), w, i), {}), (bad, (m(5, 8), m(5, 3), i), {}), (bad, (m(5, 1), w, i), {}),  # k > E
            (nb, (m(5, 8), m(5, 2, BF16), i), {}), (nb, (m(5, 8), w, m(5, 2)), {}), (nb, (m(5, 8, S8), w, i), {}),
            (nb, (m(5, 1025), w, i), {}), (nb, (m(5, 40), m(5, 33), m(5, 33, S32)), {}), (nb, (m(5, 8, F32, 1, 5), w, i), {}),
            (bad, (m(5, 8), m(5, 0), m(5, 0, S32)), {}), (nb, (m(5, 8), m(5, 2, F32, 0), i), {}), (bad, (md((5,), F32, (1,)), w, i), {}),
            (bad, (md((5, 8, 1), F32, (8, 1, 1)), w, i), {}), (bad, (m(5, 8), w, i), {"scoring": 2}), (bad, (m(5, 8), w, i), {"scoring": -1}),
            (bad, (m(5, 8), w, i), {"scale": float("nan")}), (bad, (m(5, 8), w, i), {"scale": float("inf")}),
            (bad, (md(), w, i), {}), (nb, (md.grouped((5, 8), F32, 0, 2), w, i), {}), (nb, (m(1 << 30, 8), m(1 << 30, 2), m(1 << 30, 2, S32)), {}),
            (bad, (m(O, 1), m(O, 2), m(O, 2, S32)), {})):
        refuse(status, lambda: route(api, eng, *args, **kw))
    refuse(bad, lambda: api.moe_route_backward.primitive_desc(eng, m(5, 8), i, w, m(5, 9)))
    refuse(nb, lambda: api.moe_route_backward.primitive_desc(eng, m(5, 8), i, w, m(5, 8, BF16)))
    refuse(nb, lambda: api.moe_route_backward.primitive_desc(eng, m(5, 8), i, w, m(5, 8, F32, 0)))

    g = md.grouped((10, 4), F32, 0, 8)
    for status, args in (
            (bad, (m(5, 4), i, md.grouped((9, 4), F32, 0, 8), i)), (bad, (m(5, 4), i, md.grouped((10, 5), F32, 0, 8), i)),
            (bad, (m(5, 4), i, m(10, 4), i)), (bad, (m(5, 4, BF16), i, g, i)), (bad, (m(5, 4), i, md.grouped((10, 4), F32, 1, 8), i)),
            (nb, (m(5, 4), i, md.grouped((10, 4), F32, 0, 1025), i)), (nb, (m(5, 4), m(5, 2, S64), g, i)), (bad, (m(5, 4), i, g, m(5, 3, S32))),
            (nb, (m(5, 4, 11), i, md.grouped((10, 4), 11, 0, 8), i)), (nb, (m(5, 4, S64), i, md.grouped((10, 4), S64, 0, 8), i))):
        refuse(status, lambda: api.moe_dispatch.primitive_desc(eng, *args))

    for status, args, kw in (
            (bad, (m(10, 4), i, m(5, 4)), {}), (bad, (g, i, m(4, 4)), {}), (bad, (g, i, m(5, 5)), {}), (nb, (g, i, m(5, 4, S8)), {}),
            (nb, (md.grouped((10, 4), S8, 0, 8), i, m(5, 4)), {}), (bad, (g, i, m(5, 4)), {"weights_md": m(5, 3)}),
            (nb, (g, i, m(5, 4)), {"weights_md": m(5, 2, BF16)}), (nb, (g, i, m(5, 4)), {"residual_md": m(5, 4, BF16)}),
            (bad, (g, i, m(5, 4)), {"residual_md": m(5, 5)}), (bad, (g, i, m(5, 4)), {"dropout_p": -0.1}),
            (bad, (g, i, m(5, 4)), {"dropout_p": 1.1}), (bad, (g, i, m(5, 4)), {"dropout_p": float("nan")}), (nb, (g, i, m(5, 4, F32, 0)), {})):
        refuse(status, lambda: api.moe_combine.primitive_desc(eng, *args, **kw))
    refuse(bad, lambda: api.moe_combine_backward.primitive_desc(eng, m(5, 4), g, i, w, md.grouped((10, 4), F32, 0, 7), w))
    refuse(nb, lambda: api.moe_combine_backward.primitive_desc(eng, m(5, 4), g, i, w, md.grouped((10, 4), BF16, 0, 8), w))
    refuse(bad, lambda: api.moe_combine_backward.primitive_desc(eng, m(5, 4), g, i, m(5, 3), g, w))

    refuse(bad, lambda: api.dropout.primitive_desc(eng, m(5, 4), m(5, 5), 0.1))
    refuse(nb, lambda: api.dropout.primitive_desc(eng, m(5, 4), m(5, 4, BF16), 0.1))
    refuse(nb, lambda: api.dropout.primitive_desc(eng, m(5, 4, S8), m(5, 4, S8), 0.1))
    refuse(bad, lambda: api.dropout.primitive_desc(eng, m(5, 4), m(5, 4), 1.5))
    refuse(bad, lambda: api.dropout.primitive_desc(eng, m(5, 4), m(5, 4), 0.5, residual_md=m(4, 4)))

    attr = api.primitive_attr()
    attr.set_scales_mask(api.ARG_SRC, 0)
    refuse(nb, lambda: api.dropout.primitive_desc(eng, m(5, 4), m(5, 4), 0.1, attr=attr))
    assert api.lib().dnnl_cuda_interop_dropout_primitive_desc_create(None, eng._h, m(5, 4)._h, None, m(5, 4)._h, 0.1, None) == bad


def test_execution_arguments(host_engine):
    """missing, unknown and unbacked arguments are refused before anything is launched"""
    import torch
    from onednn_b200 import api
    if torch.cuda.is_available():
        pytest.skip("for an engine without a device: the pointers lead nowhere")
    md, m = mats(api)
    prim = api.dropout(api.dropout.primitive_desc(host_engine, m(5, 4), m(5, 4), 0.5))
    strm = api.stream(host_engine)
    none = api.memory(m(5, 4), host_engine, 0)
    seed = api.memory(md((2,), S64, (1,)), host_engine, 64)
    some = api.memory(m(5, 4), host_engine, 64)
    for args in ({}, {api.ARG_SRC: some, api.ARG_DST: some}, {api.ARG_SRC: none, api.ARG_DST: some, api.ARG_ATTR_DROPOUT_SEED: seed},
                 {api.ARG_SRC: some, api.ARG_DST: some, api.ARG_ATTR_DROPOUT_SEED: seed, api.ARG_SRC_2: some}):
        with pytest.raises(api.error) as e:
            prim.execute(strm, args)
        assert e.value.status == api.invalid_arguments
    with pytest.raises(api.error) as e:  # an engine without a device
        prim.execute(strm, {api.ARG_SRC: some, api.ARG_DST: some, api.ARG_ATTR_DROPOUT_SEED: seed})
    assert e.value.status == api.runtime_error


@pytest.mark.parametrize("file", ["moe_route.cu", "moe_dispatch.cu", "moe_combine.cu", "dropout.cu"])
def test_kernels_read_with_coherent_loads_behind_their_wait(file):
    kernels = _reachable(file)
    assert kernels, "no kernel with a wait in " + file
    for name, text in kernels.items():
        assert not NON_COHERENT.findall(text), name

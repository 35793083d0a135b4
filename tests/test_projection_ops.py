"""What the operators around a quantized projection promise of one another, without a device: which of the norm's outputs the products
take and by which kernel, and when the adapters have a scratchpad."""
import os
import re

import pytest

BF16, F32, S32, S8, E4M3 = 2, 3, 4, 5, 10


@pytest.mark.parametrize("out,mask,groups,impl", [(S8, 0, (), "cuda:tcgen05:int8"), (S8, 1, (), "cuda:tcgen05:int8"), (E4M3, 0, (), "cuda:tcgen05:fp8"),
                                                  (E4M3, 1, (), None), (S8, 3, (1, 128), "cuda:ref_int8:any"), (E4M3, 3, (1, 128), "cuda:ref:any")])
def test_products_of_what_the_norm_writes(host_engine, out, mask, groups, impl):
    """the scales that the norm takes for its dst, given to the product for its src"""
    from onednn_b200 import api
    md, eng = api.memory.desc, host_engine
    T, H, N = 256, 1024, 512
    attr = api.primitive_attr()
    attr.set_scales(api.ARG_DST, mask, groups, qmode=api.quantization_mode.dynamic_fp if mask else api.quantization_mode.static_sazp)
    x, q = md((T, H), BF16, (H, 1)), md((T, H), out, (H, 1))
    norm = api.rms_norm.primitive_desc(eng, x, q, 1e-5, attr=attr)
    assert norm.query_md(255, api.ARG_ATTR_SCALES | api.ARG_DST).get_dims() == ((T if mask & 1 else 1), (H // groups[1] if groups else 1))
    attr = api.primitive_attr()
    attr.set_scales(api.ARG_SRC, mask, groups)
    attr.set_scales(api.ARG_WEIGHTS, 2)

    def product():
        return api.matmul.primitive_desc(eng, q, md((H, N), out, (N, 1)), md((T, N), F32, (N, 1)), None, attr)

    if impl is None:
        with pytest.raises(api.error) as e:
            product()
        assert e.value.status == api.unimplemented
    else:
        assert product().impl_info_str() == impl


def test_scratchpad_of_the_adapters(host_engine):
    from onednn_b200 import api
    md, O = api.memory.desc, api.RUNTIME_DIM_VAL
    attr = api.primitive_attr()
    attr.set_scratchpad_mode(api.SCRATCHPAD_MODE_USER)

    def bytes_(T, r, n=3, K=32, N=48):
        up = (O, O, 1) if r == O else (r * N, N, 1)
        pd = api.low_rank_adapter.primitive_desc(
            host_engine, md((T, K), BF16, (K, 1)), md((T,), S32, (1,)), md((n, K, r), BF16, (O, O, 1) if r == O else (K * r, r, 1)),
            md((n, r, N), BF16, up), md((T, N), BF16, (N, 1)), attr=attr)
        scratch = pd.query_md(255, api.ARG_SCRATCHPAD)
        return scratch.get_dims()[0] if scratch.get_ndims() else 0

    assert bytes_(1024, 32) == bytes_(512, 33) == bytes_(512, 128) == bytes_(512, O) == bytes_(1, 1) == 0
    assert all(bytes_(T, r) for T, r in ((1025, 1), (1025, 32), (513, 33), (513, 128), (513, O), (O, 8), (O, O)))


@pytest.mark.parametrize("file", ["rms_norm.cu", "low_rank.cu"])
def test_shared_memory_of_wide_accesses_is_aligned(file):
    """what a launch sizes stands on a 16-byte boundary by its declaration, not by what happens to lie in front of it"""
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "onednn_b200", "csrc")
    with open(os.path.join(csrc, file)) as f:
        declared = re.findall(r"extern __shared__ ([^;]*);", f.read())
    assert declared and all(d.startswith("__align__(16) ") for d in declared), declared

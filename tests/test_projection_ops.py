"""What the operators around a quantized projection promise, without a device: when the adapters have a scratchpad."""
BF16, S32 = 2, 4


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

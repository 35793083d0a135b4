"""A mixture-of-experts layer on the library's primitives, forward and the router's way back.

    python examples/moe_layer.py [--tokens 512] [--hidden 1024] [--inner 2048] [--experts 16] [--choices 4] [--dropout 0.1]

    logits   = x W_r                              matmul, s8 weights
    w, idx   = the best `choices` of the logits   moe_route
    rows     = x sorted by expert                 moe_dispatch: grouped memory, made on the device
    inner    = swish(rows W_1[expert])            matmul on grouped memory, s8 weights
    out      = inner W_2[expert]                  matmul on grouped memory, s8 weights
    y        = x + dropout(sum w out)             moe_combine

and from a gradient of y the gradients of the experts' results and of w (moe_combine_backward) and of the logits
(moe_route_backward): what trains the router beside frozen quantized experts.  The experts' own way back, from their results
to the tokens, is not part of it.  Nothing waits on the host in between: one stream, no copies.  The results are compared
with plain torch in 32 bits.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from onednn_b200 import api  # noqa: E402

F16, BF16, F32, S32, S8, S64 = 1, 2, 3, 4, 5, 16
_CODE = {torch.bfloat16: BF16, torch.float32: F32, torch.int32: S32, torch.int8: S8, torch.int64: S64}
ELTWISE_SWISH = 0x2c


class Step:
    """One primitive and the memory objects behind its arguments."""

    def __init__(self, layer):
        self.layer, self.args, self.keep = layer, {}, []

    def mem(self, arg, t):
        md = api.memory.desc(tuple(t.shape), _CODE[t.dtype], tuple(t.stride()))
        self.args[arg] = api.memory(md, self.layer.eng, t.data_ptr())
        self.keep.append(t)
        return md

    def grouped(self, arg, t):
        md = api.memory.desc.grouped(tuple(t.shape), _CODE[t.dtype], 0, self.layer.experts)
        self.args[arg] = api.memory(md, self.layer.eng, handles=[t.data_ptr(), self.layer.offsets.data_ptr()])
        self.keep.append(t)
        return md

    def done(self, primitive, *pd_args, **pd_kw):
        self.prim = primitive(primitive.primitive_desc(self.layer.eng, *pd_args, **pd_kw))
        return self

    def __call__(self):
        self.prim.execute(self.layer.strm, self.args)


class MoeLayer:
    def __init__(self, tokens, hidden, inner, experts, choices, dropout, seed=1):
        self.eng = api.engine(api.engine.kind.gpu, torch.cuda.current_device())
        self.strm = api.stream(self.eng, torch.cuda.current_stream().cuda_stream)
        self.experts, self.choices, self.p = experts, choices, dropout
        g = torch.Generator(device="cuda").manual_seed(seed)

        def weights(*shape):  # s8 values, and a scale per (expert,) column
            w = torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=torch.int8)
            scale = (torch.rand(shape[:-2] + (1, shape[-1]), generator=g, device="cuda") + 0.5) / (127 * shape[-2] ** 0.5)
            return w, scale

        self.w_router, self.w_in, self.w_out = weights(hidden, experts), weights(experts, hidden, inner), weights(experts, inner, hidden)

        def empty(*shape, dtype=torch.bfloat16):
            return torch.empty(shape, device="cuda", dtype=dtype)

        n = tokens * choices
        self.x, self.y, self.dy = empty(tokens, hidden), empty(tokens, hidden), empty(tokens, hidden)
        self.logits, self.w = empty(tokens, experts, dtype=torch.float32), empty(tokens, choices, dtype=torch.float32)
        self.idx, self.pos = empty(tokens, choices, dtype=torch.int32), empty(tokens, choices, dtype=torch.int32)
        self.offsets = empty(experts, dtype=torch.int32)
        self.rows, self.inner, self.out, self.drows = empty(n, hidden), empty(n, inner), empty(n, hidden), empty(n, hidden)
        self.dw, self.dlogits = torch.empty_like(self.w), torch.empty_like(self.logits)
        self.seed = torch.tensor([20240607, 0], dtype=torch.int64, device="cuda")  # (seed, offset): the offset counts steps

        attr = api.primitive_attr()
        attr.set_fpmath_mode(api.fpmath_mode.bf16, True)
        attr.set_scales(api.ARG_WEIGHTS, 2, (), F32)
        s = self.product = Step(self)
        s.mem(api.ARG_ATTR_SCALES | api.ARG_WEIGHTS, self.w_router[1])
        s.done(api.matmul, s.mem(api.ARG_SRC, self.x), s.mem(api.ARG_WEIGHTS, self.w_router[0]), s.mem(api.ARG_DST, self.logits), None, attr)

        s = self.route = Step(self)
        s.done(api.moe_route, s.mem(api.ARG_SRC, self.logits), s.mem(api.ARG_DST, self.w), s.mem(api.ARG_DST_1, self.idx), normalize=True)

        s = self.dispatch = Step(self)
        s.done(api.moe_dispatch, s.mem(api.ARG_SRC, self.x), s.mem(api.ARG_SRC_1, self.idx), s.grouped(api.ARG_DST, self.rows),
               s.mem(api.ARG_DST_1, self.pos))

        def expert(src, w, dst, swish):
            attr = api.primitive_attr()
            attr.set_fpmath_mode(api.fpmath_mode.bf16, True)
            attr.set_scales(api.ARG_WEIGHTS, 0b101, (), F32)
            if swish:
                po = api.post_ops()
                po.append_eltwise(ELTWISE_SWISH, 1.0, 0.0)
                attr.set_post_ops(po)
            s = Step(self)
            s.mem(api.ARG_ATTR_SCALES | api.ARG_WEIGHTS, w[1])
            return s.done(api.matmul, s.grouped(api.ARG_SRC, src), s.mem(api.ARG_WEIGHTS, w[0]), s.grouped(api.ARG_DST, dst), None, attr)

        self.up, self.down = expert(self.rows, self.w_in, self.inner, True), expert(self.inner, self.w_out, self.out, False)

        s = self.combine = Step(self)
        if dropout:
            s.mem(api.ARG_ATTR_DROPOUT_SEED, self.seed)
        s.done(api.moe_combine, s.grouped(api.ARG_SRC, self.out), s.mem(api.ARG_SRC_1, self.pos), s.mem(api.ARG_DST, self.y),
               weights_md=s.mem(api.ARG_WEIGHTS, self.w), residual_md=s.mem(api.ARG_SRC_2, self.x), dropout_p=dropout)

        s = self.combine_grad = Step(self)
        if dropout:
            s.mem(api.ARG_ATTR_DROPOUT_SEED, self.seed)
        s.done(api.moe_combine_backward, s.mem(api.ARG_DIFF_DST, self.dy), s.grouped(api.ARG_SRC, self.out),
               s.mem(api.ARG_SRC_1, self.pos), s.mem(api.ARG_WEIGHTS, self.w), s.grouped(api.ARG_DIFF_SRC, self.drows),
               s.mem(api.ARG_DIFF_WEIGHTS, self.dw), dropout_p=dropout)

        s = self.route_grad = Step(self)
        s.done(api.moe_route_backward, s.mem(api.ARG_SRC, self.logits), s.mem(api.ARG_SRC_1, self.idx), s.mem(api.ARG_DIFF_DST, self.dw),
               s.mem(api.ARG_DIFF_SRC, self.dlogits), normalize=True)

    def forward(self):
        for step in (self.product, self.route, self.dispatch, self.up, self.down, self.combine):
            step()

    def backward(self):
        for step in (self.combine_grad, self.route_grad):
            step()

    def plain(self):
        """(y, dw, dlogits, gradient of the experts' results by slot) in 32 bits, from the layer's own choices and mask; the
        experts' rows rounded as they are stored"""
        x, idx, bf = self.x.float(), self.idx.long(), lambda t: t.bfloat16().float()
        logits = (x @ (self.w_router[0].float() * self.w_router[1])).requires_grad_()
        w = torch.softmax(torch.gather(logits, 1, idx), 1)
        terms = torch.zeros(idx.shape + (x.shape[1],), device="cuda")
        for e in range(self.experts):
            t, j = torch.nonzero(idx == e, as_tuple=True)
            h = bf(torch.nn.functional.silu(x[t] @ (self.w_in[0][e].float() * self.w_in[1][e])))
            terms[t, j] = bf(h @ (self.w_out[0][e].float() * self.w_out[1][e]))
        terms.requires_grad_()
        w.retain_grad()
        kept = torch.ones_like(x)
        if self.p:  # the mask: dropout of ones
            s, ones = Step(self), torch.ones_like(x)
            s.mem(api.ARG_ATTR_DROPOUT_SEED, self.seed)
            s.done(api.dropout, s.mem(api.ARG_SRC, ones), s.mem(api.ARG_DST, kept), self.p)()
        y = x + (w.unsqueeze(2) * terms).sum(1) * kept
        y.backward(self.dy.float())
        return y.detach(), w.grad, logits.grad, terms.grad


def run(tokens=512, hidden=1024, inner=2048, experts=16, choices=4, dropout=0.1):
    """Largest differences from the plain form, relative to its largest values."""
    layer = MoeLayer(tokens, hidden, inner, experts, choices, dropout)
    layer.x.normal_()
    layer.dy.normal_()
    layer.seed[1] += 1
    layer.forward()
    layer.backward()
    layer.strm.wait()
    results = {"y": layer.y, "dw": layer.dw, "dlogits": layer.dlogits, "drows": layer.drows[layer.pos.long()]}
    result = {name: ((got.float() - want).abs().max() / want.abs().max()).item()
              for (name, got), want in zip(results.items(), layer.plain())}
    return result, layer


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    for name, value in (("tokens", 512), ("hidden", 1024), ("inner", 2048), ("experts", 16), ("choices", 4), ("dropout", 0.1)):
        ap.add_argument("--" + name, type=type(value), default=value)
    difference, layer = run(**vars(ap.parse_args()))
    print("rows per expert:", layer.offsets.diff(prepend=layer.offsets.new_zeros(1)).tolist())
    print("differences from the plain form:", difference)
    assert max(difference.values()) < 0.02

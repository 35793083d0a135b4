"""A quantized projection with adapters of many requests, and the router of a layer behind it, forward and the tokens' way back.

    python examples/adapted_projection.py [--tokens 384] [--hidden 1024] [--outputs 1536] [--rank 16] [--adapters 6] [--experts 64]

    h, q, s = norm of x + residual                 rms_norm: the sum, s8 values and a scale for each token
    y       = (s q) W                              matmul, s8 x s8
    y_t     = y_t + scale_i (n_t A_i) B_i          low_rank_adapter, in place: i is the adapter of token t's request, n the norm in bf16
    w, e    = the best experts of logits + bias    moe_route, within the best groups of experts

and from gradients of y and of h the gradient of x and of the norm's weights: the adapters' share (low_rank_adapter with the
factors exchanged, on top of the frozen projection's own, which is given here) and the norm's (rms_norm_backward).  One stream, no
copies, no waits in between.  The results are compared with plain torch in 32 bits.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from onednn_b200 import api  # noqa: E402

_CODE = {torch.bfloat16: 2, torch.float32: 3, torch.int32: 4, torch.int8: 5}
EPSILON = 1e-5


class Step:
    """One primitive and the memory objects behind its arguments."""

    def __init__(self, layer):
        self.layer, self.args, self.keep = layer, {}, []

    def mem(self, arg, t):
        md = api.memory.desc(tuple(t.shape), _CODE[t.dtype], tuple(t.stride()))
        self.args[arg] = api.memory(md, self.layer.eng, t.data_ptr())
        self.keep.append(t)
        return md

    def done(self, primitive, *pd_args, **pd_kw):
        self.prim = primitive(primitive.primitive_desc(self.layer.eng, *pd_args, **pd_kw))
        return self

    def __call__(self):
        self.prim.execute(self.layer.strm, self.args)


class AdaptedProjection:
    def __init__(self, tokens, hidden, outputs, rank, adapters, experts, seed=1):
        self.eng = api.engine(api.engine.kind.gpu, torch.cuda.current_device())
        self.strm = api.stream(self.eng, torch.cuda.current_stream().cuda_stream)
        g = torch.Generator(device="cuda").manual_seed(seed)

        def normal(*shape, scale=1.0, dtype=torch.bfloat16):
            return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)

        def empty(*shape, dtype=torch.bfloat16):
            return torch.empty(shape, device="cuda", dtype=dtype)

        self.x, self.residual = normal(tokens, hidden), normal(tokens, hidden)
        self.gamma = 1 + normal(hidden, scale=0.1, dtype=torch.float32)
        self.sum, self.norm = empty(tokens, hidden), empty(tokens, hidden)
        self.q, self.scales = empty(tokens, hidden, dtype=torch.int8), empty(tokens, 1, dtype=torch.float32)
        self.weights = torch.randint(-127, 128, (hidden, outputs), generator=g, device="cuda", dtype=torch.int8)
        self.wscale = (torch.rand(outputs, generator=g, device="cuda") + 0.5) / (127 * hidden ** 0.5)
        self.y = empty(tokens, outputs)
        # the factors as the two layers' weights [outputs, inputs]; tokens of a request follow one another, some have no adapter
        self.down = normal(adapters, rank, hidden, scale=hidden ** -0.5).transpose(1, 2)
        self.up = normal(adapters, outputs, rank, scale=rank ** -0.5).transpose(1, 2)
        self.adapter_scale = torch.rand(adapters, generator=g, device="cuda") + 0.5
        self.index = (torch.arange(tokens, device="cuda") * (adapters + 1) // tokens - 1).to(torch.int32)
        self.logits, self.bias = normal(tokens, experts, dtype=torch.float32), normal(experts, scale=0.1, dtype=torch.float32)
        self.w, self.experts = empty(tokens, 4, dtype=torch.float32), empty(tokens, 4, dtype=torch.int32)
        # the way back: gradients of y and of the sum, and the projection's own gradient of the norm
        self.dy, self.dsum, self.dproj = normal(tokens, outputs), normal(tokens, hidden), normal(tokens, hidden)
        self.dnorm, self.dx, self.dgamma = empty(tokens, hidden), empty(tokens, hidden), empty(hidden, dtype=torch.float32)

        s = self.norm_plain = Step(self)
        s.done(api.rms_norm, s.mem(api.ARG_SRC, self.x), s.mem(api.ARG_DST, self.norm), EPSILON, weights_md=s.mem(api.ARG_WEIGHTS, self.gamma),
               residual_md=s.mem(api.ARG_SRC_2, self.residual), sum_md=s.mem(api.ARG_DST_1, self.sum))

        attr = api.primitive_attr()
        attr.set_scales(api.ARG_DST, 1, qmode=api.quantization_mode.dynamic_fp)
        s = self.quantize = Step(self)
        s.mem(api.ARG_ATTR_SCALES | api.ARG_DST, self.scales)
        s.done(api.rms_norm, s.mem(api.ARG_SRC, self.x), s.mem(api.ARG_DST, self.q), EPSILON, weights_md=s.mem(api.ARG_WEIGHTS, self.gamma),
               residual_md=s.mem(api.ARG_SRC_2, self.residual), attr=attr)

        attr = api.primitive_attr()
        attr.set_scales(api.ARG_SRC, 1)
        attr.set_scales(api.ARG_WEIGHTS, 2)
        s = self.project = Step(self)
        s.mem(api.ARG_ATTR_SCALES | api.ARG_SRC, self.scales)
        s.mem(api.ARG_ATTR_SCALES | api.ARG_WEIGHTS, self.wscale)
        s.done(api.matmul, s.mem(api.ARG_SRC, self.q), s.mem(api.ARG_WEIGHTS, self.weights), s.mem(api.ARG_DST, self.y), None, attr)

        def adapters_step(src, down, up, base, dst):
            attr = api.primitive_attr()
            attr.set_scales(api.ARG_WEIGHTS, 1)
            s = Step(self)
            s.mem(api.ARG_ATTR_SCALES | api.ARG_WEIGHTS, self.adapter_scale)
            return s.done(api.low_rank_adapter, s.mem(api.ARG_SRC, src), s.mem(api.ARG_SRC_1, self.index), s.mem(api.ARG_WEIGHTS, down),
                          s.mem(api.ARG_WEIGHTS_1, up), s.mem(api.ARG_DST, dst), base_md=s.mem(api.ARG_SRC_2, base), attr=attr)

        self.adapt = adapters_step(self.norm, self.down, self.up, self.y, self.y)
        s = self.route = Step(self)
        s.done(api.moe_route, s.mem(api.ARG_SRC, self.logits), s.mem(api.ARG_DST, self.w), s.mem(api.ARG_DST_1, self.experts),
               scoring=api.scoring.sigmoid, bias_md=s.mem(api.ARG_BIAS, self.bias), groups=8, groups_kept=2, group_best=2)

        self.adapt_grad = adapters_step(self.dy, self.up.transpose(1, 2), self.down.transpose(1, 2), self.dproj, self.dnorm)
        s = self.norm_grad = Step(self)
        s.done(api.rms_norm_backward, s.mem(api.ARG_DIFF_DST, self.dnorm), s.mem(api.ARG_SRC, self.sum), s.mem(api.ARG_DIFF_SRC, self.dx), EPSILON,
               weights_md=s.mem(api.ARG_WEIGHTS, self.gamma), diff_weights_md=s.mem(api.ARG_DIFF_WEIGHTS, self.dgamma),
               diff_sum_md=s.mem(api.ARG_SRC_2, self.dsum))

    def forward(self):
        for step in (self.norm_plain, self.quantize, self.project, self.adapt, self.route):
            step()

    def backward(self):
        for step in (self.adapt_grad, self.norm_grad):
            step()

    def plain(self):
        """(sum, y, dx, dgamma, weights of the library's choices) in 32 bits; the norm rounded as it is stored"""
        x, gamma = self.x.float().requires_grad_(), self.gamma.clone().requires_grad_()
        h = x + self.residual.float()
        n = h * torch.rsqrt((h * h).mean(1, keepdim=True) + EPSILON) * gamma
        delta = torch.zeros_like(self.y, dtype=torch.float32)
        for i in range(self.down.shape[0]):
            on = (self.index == i).nonzero()[:, 0]
            m = n[on] + (n[on].bfloat16().float() - n[on]).detach()
            delta = delta.index_add(0, on, self.adapter_scale[i] * (m @ self.down[i].float()) @ self.up[i].float())
        y = self.q.float() * self.scales @ (self.weights.float() * self.wscale) + delta
        (h * self.dsum.float() + n * self.dproj.float()).sum().add((delta * self.dy.float()).sum()).backward()
        s = torch.sigmoid(torch.gather(self.logits, 1, self.experts.long()))
        return h.detach(), y.detach(), x.grad, gamma.grad, s / s.sum(1, keepdim=True)


def run(tokens=384, hidden=1024, outputs=1536, rank=16, adapters=6, experts=64):
    """Largest differences from the plain form, relative to its largest values."""
    layer = AdaptedProjection(tokens, hidden, outputs, rank, adapters, experts)
    layer.forward()
    layer.backward()
    layer.strm.wait()
    results = {"sum": layer.sum, "y": layer.y, "dx": layer.dx, "dgamma": layer.dgamma, "w": layer.w}
    return {name: ((got.float() - want).abs().max() / want.abs().max()).item() for (name, got), want in zip(results.items(), layer.plain())}, layer


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    for name, value in (("tokens", 384), ("hidden", 1024), ("outputs", 1536), ("rank", 16), ("adapters", 6), ("experts", 64)):
        ap.add_argument("--" + name, type=int, default=value)
    difference, layer = run(**vars(ap.parse_args()))
    print("tokens per adapter:", torch.bincount(layer.index.clamp_min(-1).long() + 1).tolist()[1:])
    print("differences from the plain form:", difference)
    assert max(difference.values()) < 0.02

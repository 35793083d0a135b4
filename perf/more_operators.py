"""Performance cases of the operators around a quantized projection: the norm that makes its 8-bit operand, the low-rank
adapters beside it, and the router with a bias and groups of experts.

The products themselves are ``dnnl::matmul`` (``perf/cases.py``); the plain router, the sort into grouped rows and the way
back are in ``perf/operators.py``.

``op`` of a case
  norm        x (+ residual, whose sum is written) -> its root-mean-square norm times gamma, in 16 or 32 bits, or in 8 bits
              with one given scale ("tensor"), or with scales that are made per row ("row") or per group of a row ("group")
  norm_grad   gradients of that: of the sum (with what comes along the residual path), and of gamma
  route       logits -> the k experts of each token, chosen by score + bias within the best groups, and their weights
  adapters    base + scale[i] (x A[i]) B[i], i the adapter of each row (or none)
"""
import math

import numpy as np
import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "s8": torch.int8, "e4m3": torch.float8_e4m3fn}
_CODE = {"f16": 1, "bf16": 2, "f32": 3, "s32": 4, "s8": 5, "e4m3": 10}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2, "s8": 1, "e4m3": 1}
_LIMIT = {"s8": 127.0, "e4m3": 448.0}
EPS = 1e-5


def listed():
    return [
        # token generation, one sequence: the norm in front of an fp8 projection with a calibrated scale (latency)
        {"name": "norm_token", "op": "norm", "T": 1, "H": 4096, "dtype": "bf16", "out": "e4m3", "scales": "tensor", "group": 0,
         "residual": True, "gamma": "bf16", "pitch": 0},
        # a full batch of prompts in front of an fp8 projection
        {"name": "norm_prefill", "op": "norm", "T": 8192, "H": 4096, "dtype": "bf16", "out": "e4m3", "scales": "tensor",
         "group": 0, "residual": True, "gamma": "bf16", "pitch": 0},
        # the operand of an int8 projection with a scale a row, made from the row
        {"name": "norm_row_scales", "op": "norm", "T": 2048, "H": 5120, "dtype": "bf16", "out": "s8", "scales": "row", "group": 0,
         "residual": True, "gamma": "f32", "pitch": 0},
        # scales of 128 columns each, a batch of an odd size
        {"name": "norm_group_scales", "op": "norm", "T": 4099, "H": 4096, "dtype": "bf16", "out": "e4m3", "scales": "group",
         "group": 128, "residual": False, "gamma": "bf16", "pitch": 0},
        # an odd width inside a wider buffer, no quantization
        {"name": "norm_ragged", "op": "norm", "T": 3001, "H": 2047, "dtype": "f16", "out": "f16", "scales": "", "group": 0,
         "residual": True, "gamma": "f16", "pitch": 2053},
        # training step, backward, with the gradient that comes along the residual path
        {"name": "norm_grad", "op": "norm_grad", "T": 8192, "H": 4096, "dtype": "bf16", "residual": True, "gamma": "bf16",
         "pitch": 0},
        # backward in 32 bits, an odd width inside a wider buffer
        {"name": "norm_grad_f32", "op": "norm_grad", "T": 1021, "H": 1367, "dtype": "f32", "residual": False, "gamma": "f32",
         "pitch": 1371},
        # token generation, one sequence: the router of a 256-expert layer in eight groups
        {"name": "route_token", "op": "route", "T": 1, "E": 256, "k": 8, "dtype": "f32", "scoring": "sigmoid", "bias": True,
         "groups": 8, "kept": 4, "best": 2, "normalize": True, "scale": 2.5},
        # a full batch of prompts
        {"name": "route_prefill", "op": "route", "T": 8192, "E": 256, "k": 8, "dtype": "f32", "scoring": "sigmoid", "bias": True,
         "groups": 8, "kept": 4, "best": 2, "normalize": True, "scale": 2.5},
        # token generation, a batch of sequences of many customers: every row has an adapter of its own choice
        {"name": "adapters_decode", "op": "adapters", "T": 61, "n": 64, "K": 4096, "N": 4096, "r": 16, "dtype": "bf16",
         "out": "bf16", "base": True, "order": "mixed", "none": 0.05, "layout": "out_in", "pitch": 0},
        # a full batch of prompts of sixteen adapters beside a wide projection: the largest case
        {"name": "adapters_prefill", "op": "adapters", "T": 8192, "n": 16, "K": 4096, "N": 11008, "r": 32, "dtype": "bf16",
         "out": "bf16", "base": True, "order": "requests", "none": 0.1, "layout": "out_in", "pitch": 0},
        # rows of several requests in any order, other layouts and types, an odd batch
        {"name": "adapters_mixed", "op": "adapters", "T": 777, "n": 37, "K": 2048, "N": 5504, "r": 8, "dtype": "f16",
         "out": "f32", "base": False, "order": "mixed", "none": 0.1, "layout": "in_out", "pitch": 0},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo=64, hi=8192):
    """Three of four widths are multiples of 64, as layers are; the others any number, odd ones among them."""
    h = _log_int(rng, lo, hi)
    return max(64, h // 64 * 64) if rng.random() < 0.75 else h


def draw(rng):
    op = rng.choice(["norm", "norm", "norm_grad", "route", "adapters", "adapters"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op.startswith("norm"):
        t, h = _log_int(rng, 1, 16384), _width(rng)
        while t * h * _SIZE[dtype] > 8192 * 4096 * 2:
            t = max(1, t // 2)
        c = {"op": op, "T": t, "H": h, "dtype": dtype, "residual": rng.random() < 0.6, "gamma": rng.choice([dtype, "f32"]),
             "pitch": h + rng.randint(1, 64) if rng.random() < 0.2 else 0}
        if op == "norm":
            c["out"] = rng.choice([dtype, "s8", "e4m3", "e4m3"])
            c["scales"], c["group"] = "", 0
            if c["out"] in _LIMIT:
                c["scales"] = rng.choice(["tensor", "row", "group"])
            if c["scales"] == "group":
                c["group"] = rng.choice([32, 64, 128])
                c["H"] = max(c["group"], h // c["group"] * c["group"])
                c["pitch"] = c["H"] + c["pitch"] - h if c["pitch"] else 0
        return c
    if op == "route":
        groups = rng.choice([1, 2, 4, 8, 8, 16])
        size = _log_int(rng, 2, max(2, min(64, 512 // groups)))
        kept = rng.randint(1, groups)
        k = min(kept * size, rng.choice([1, 2, 4, 6, 8]))
        return {"op": op, "T": _log_int(rng, 1, 16384), "E": groups * size, "k": k, "dtype": dtype,
                "scoring": rng.choice(["softmax", "sigmoid"]), "bias": groups == 1 or rng.random() < 0.7, "groups": groups, "kept": kept,
                "best": rng.choice([1, 2]), "normalize": rng.random() < 0.7, "scale": rng.choice([1.0, 2.5])}
    dtype = rng.choice(["bf16", "bf16", "f16"])
    t, n, k, m = _log_int(rng, 1, 8192), _log_int(rng, 1, 64), _width(rng, 128, 8192), _width(rng, 128, 11008)
    r = rng.choice([4, 8, 8, 16, 16, 32, 64, 12, 24])
    while n > 1 and n * r > 512:
        n //= 2
    while t > 1 and t * (k + 2 * m) > 8192 * (4096 + 2 * 4096):
        t //= 2
    return {"op": op, "T": t, "n": n, "K": k, "N": m, "r": r, "dtype": dtype, "out": rng.choice([dtype, dtype, "f32"]),
            "base": rng.random() < 0.8, "order": rng.choice(["requests", "mixed"]), "none": rng.choice([0.0, 0.1, 0.5]),
            "layout": rng.choice(["out_in", "in_out"]), "pitch": m + rng.randint(1, 64) if rng.random() < 0.15 else 0}


# ---------------------------------------------------------------------------------------------------- inputs


def _rows(g, shape, dtype, pitch=0, scale=1.0):
    """A matrix of normal values, with `pitch` elements from row to row where that is given."""
    m, n = shape
    return (torch.randn((m, pitch or n), generator=g, device="cuda") * scale).to(_DT[dtype])[:, :n]


def _inputs(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op, s = case["op"], {}
    if op.startswith("norm"):
        t, h = case["T"], case["H"]
        # rows of a residual stream differ in size, and a few of its columns are much larger than the others
        size = torch.exp(0.5 * torch.randn((t, 1), generator=g, device="cuda"))
        loud = 1.0 + 9.0 * (torch.rand(h, generator=g, device="cuda") < 0.005)

        def stream(scale):
            m = torch.empty((t, case["pitch"] or h), device="cuda", dtype=_DT[case["dtype"]])[:, :h]
            return m.copy_(torch.randn((t, h), generator=g, device="cuda") * size * loud * scale)

        s["gamma"] = (1.0 + 0.2 * torch.randn(h, generator=g, device="cuda")).to(_DT[case["gamma"]])
        if op == "norm":
            s["x"] = stream(0.5 if case["residual"] else 1.0)
            if case["residual"]:
                s["residual"] = stream(1.0)
            if case["scales"] == "tensor":  # calibrated: most values fit, the largest saturate
                s["scale"] = torch.rand(1, generator=g, device="cuda") * 0.2 / _LIMIT[case["out"]] + 8.0 / _LIMIT[case["out"]]
        else:
            s["h"] = stream(1.0)
            s["dy"] = _rows(g, (t, h), case["dtype"], case["pitch"])
            if case["residual"]:
                s["dsum"] = _rows(g, (t, h), case["dtype"])
        return s
    if op == "route":
        demand = torch.randn(case["E"], generator=g, device="cuda") * 0.5
        s["logits"] = (torch.randn((case["T"], case["E"]), generator=g, device="cuda") + demand).to(_DT[case["dtype"]])
        if case["bias"]:  # what balances the demand, up to its last steps
            slope = 0.25 if case["scoring"] == "sigmoid" else 1.0 / case["E"]
            s["bias"] = slope * (0.05 * torch.randn(case["E"], generator=g, device="cuda") - demand)
        return s
    t, n, k, m, r = (case[v] for v in ("T", "n", "K", "N", "r"))
    s["x"] = _rows(g, (t, k), case["dtype"])
    down = torch.randn((n, r, k) if case["layout"] == "out_in" else (n, k, r), generator=g, device="cuda") * k ** -0.5
    up = torch.randn((n, m, r) if case["layout"] == "out_in" else (n, r, m), generator=g, device="cuda") * r ** -0.5
    down, up = down.to(_DT[case["dtype"]]), up.to(_DT[case["dtype"]])
    if case["layout"] == "out_in":  # stored as the two layers' weights [outputs, inputs]
        down, up = down.transpose(1, 2), up.transpose(1, 2)
    s["down"], s["up"] = down, up
    s["scale"] = 0.5 + torch.rand(n, generator=g, device="cuda")
    if case["order"] == "mixed":
        index = torch.randint(0, n, (t,), generator=g, device="cuda")
        none = torch.rand(t, generator=g, device="cuda") < case["none"]
    else:  # neighbouring rows are one request's
        requests = max(1, min(t, 3 * n // 2))
        cuts = torch.sort(torch.randint(0, t, (requests - 1,), generator=g, device="cuda")).values
        request = torch.searchsorted(cuts, torch.arange(t, device="cuda"), right=True)
        index = torch.randint(0, n, (requests,), generator=g, device="cuda")[request]
        none = (torch.rand(requests, generator=g, device="cuda") < case["none"])[request]
    s["index"] = torch.where(none, -1, index).to(torch.int32)
    if case["base"]:
        s["base"] = _rows(g, (t, m), case["out"], case["pitch"])
    return s


# ------------------------------------------------------------------------------- the framework's operators


class _Call:
    """One primitive with the memory objects that wrap the program's device buffers."""

    def __init__(self):
        from onednn_b200 import api
        self.api = api
        self.eng = api.engine(api.engine.kind.gpu, torch.cuda.current_device())
        self.strm = api.stream(self.eng, torch.cuda.current_stream().cuda_stream)
        self.args, self.keep, self.after = {}, [], None

    def bind(self, arg, t):
        names = {torch.float32: "f32", torch.bfloat16: "bf16", torch.float16: "f16", torch.int32: "s32", torch.int8: "s8",
                 torch.float8_e4m3fn: "e4m3"}
        md = self.api.memory.desc(tuple(t.shape), _CODE[names[t.dtype]], tuple(t.stride()))
        self.args[arg] = self.api.memory(md, self.eng, t.data_ptr())
        self.keep.append(t)
        return md

    def make(self, primitive, pd, outputs):
        self.prim, self.outputs = primitive(pd), outputs
        return self

    def __call__(self):
        self.prim.execute(self.strm, self.args)
        return self.outputs if self.after is None else self.after(self.outputs)


def _empty(shape, dtype):
    return torch.empty(shape, device="cuda", dtype=dtype)


def _whole(out):
    """s8 values are returned in 16 bits, which hold them exactly"""
    return (out[0].to(torch.bfloat16),) + tuple(out[1:])


def _prepare_own(case, s):
    c = _Call()
    api, op = c.api, case["op"]
    if op == "norm":
        t, h = case["T"], case["H"]
        outputs = [_empty((t, h), _DT[case["out"]])]
        attr = residual = total = None
        if case["scales"]:
            attr = api.primitive_attr()
            mode = api.quantization_mode
            if case["scales"] == "tensor":
                attr.set_scales(api.ARG_DST, 0)
                scale = s["scale"]
            elif case["scales"] == "row":
                attr.set_scales(api.ARG_DST, 1, qmode=mode.dynamic_fp)
                scale = _empty((t, 1), torch.float32)
            else:
                attr.set_scales(api.ARG_DST, 3, (1, case["group"]), qmode=mode.dynamic_fp)
                scale = _empty((t, h // case["group"]), torch.float32)
            c.bind(api.ARG_ATTR_SCALES | api.ARG_DST, scale)
            if case["scales"] != "tensor":
                outputs.append(scale)
        if case["residual"]:
            outputs.append(_empty((t, h), _DT[case["dtype"]]))
            residual, total = c.bind(api.ARG_SRC_2, s["residual"]), c.bind(api.ARG_DST_1, outputs[-1])
        pd = api.rms_norm.primitive_desc(c.eng, c.bind(api.ARG_SRC, s["x"]), c.bind(api.ARG_DST, outputs[0]), EPS,
                                         weights_md=c.bind(api.ARG_WEIGHTS, s["gamma"]), residual_md=residual, sum_md=total,
                                         attr=attr)
        c.after = _whole if case["out"] == "s8" else None
        return c.make(api.rms_norm, pd, tuple(outputs))
    if op == "norm_grad":
        dh, dgamma = _empty((case["T"], case["H"]), _DT[case["dtype"]]), _empty((case["H"],), torch.float32)
        pd = api.rms_norm_backward.primitive_desc(
            c.eng, c.bind(api.ARG_DIFF_DST, s["dy"]), c.bind(api.ARG_SRC, s["h"]), c.bind(api.ARG_DIFF_SRC, dh), EPS,
            weights_md=c.bind(api.ARG_WEIGHTS, s["gamma"]), diff_weights_md=c.bind(api.ARG_DIFF_WEIGHTS, dgamma),
            diff_sum_md=c.bind(api.ARG_SRC_2, s["dsum"]) if case["residual"] else None)
        return c.make(api.rms_norm_backward, pd, (dh, dgamma))
    if op == "route":
        w, i = _empty((case["T"], case["k"]), torch.float32), _empty((case["T"], case["k"]), torch.int32)
        pd = api.moe_route.primitive_desc(
            c.eng, c.bind(api.ARG_SRC, s["logits"]), c.bind(api.ARG_DST, w), c.bind(api.ARG_DST_1, i),
            scoring=getattr(api.scoring, case["scoring"]), normalize=case["normalize"], scale=case["scale"],
            bias_md=c.bind(api.ARG_BIAS, s["bias"]) if case["bias"] else None, groups=case["groups"],
            groups_kept=case["kept"], group_best=case["best"])
        return c.make(api.moe_route, pd, (w, i))
    y = _empty((case["T"], case["N"]), _DT[case["out"]])
    attr = api.primitive_attr()
    attr.set_scales(api.ARG_WEIGHTS, 1)
    c.bind(api.ARG_ATTR_SCALES | api.ARG_WEIGHTS, s["scale"])
    pd = api.low_rank_adapter.primitive_desc(
        c.eng, c.bind(api.ARG_SRC, s["x"]), c.bind(api.ARG_SRC_1, s["index"]), c.bind(api.ARG_WEIGHTS, s["down"]),
        c.bind(api.ARG_WEIGHTS_1, s["up"]), c.bind(api.ARG_DST, y),
        base_md=c.bind(api.ARG_SRC_2, s["base"]) if case["base"] else None, attr=attr)
    return c.make(api.low_rank_adapter, pd, y)


# ------------------------------------------------------------------------------------------- plain forms


def _eight_bits(y, out):
    limit = _LIMIT[out]
    if out == "s8":
        return torch.round(y).clamp(-limit - 1, limit).to(torch.bfloat16)
    return y.clamp(-limit, limit).to(torch.float8_e4m3fn)


def _plain(case, s):
    op = case["op"]
    if op == "norm":
        h = s["x"].float()
        if case["residual"]:
            h = h + s["residual"].float()
        y = h * torch.rsqrt((h * h).mean(1, keepdim=True) + EPS) * s["gamma"].float()
        total = (h.to(_DT[case["dtype"]]),) if case["residual"] else ()
        if not case["scales"]:
            return (y.to(_DT[case["out"]]),) + total
        if case["scales"] == "tensor":
            return (_eight_bits(y / s["scale"], case["out"]),) + total
        parts = y.view(case["T"], -1, case["group"] or case["H"])
        scale = parts.abs().amax(2) / _LIMIT[case["out"]]
        y = (parts / scale.unsqueeze(2)).view(y.shape)
        return (_eight_bits(y, case["out"]), scale) + total
    if op == "norm_grad":
        h, dy = s["h"].float(), s["dy"].float()
        r = torch.rsqrt((h * h).mean(1, keepdim=True) + EPS)
        z = dy * s["gamma"].float()
        dh = r * z - h * r ** 3 * (h * z).mean(1, keepdim=True)
        if case["residual"]:
            dh = dh + s["dsum"].float()
        return dh.to(_DT[case["dtype"]]), (dy * h * r).double().sum(0).float()
    if op == "route":
        l = s["logits"].double()  # the choice falls between neighbouring values
        if case["scoring"] == "sigmoid":
            score = 1.0 / (1.0 + torch.exp(-l))
        else:
            e = torch.exp(l - l.amax(1, keepdim=True))
            score = e / e.sum(1, keepdim=True)
        c = score + s["bias"].double() if case["bias"] else score
        if case["groups"] > 1:
            grouped = c.view(case["T"], case["groups"], -1)
            best = torch.sort(grouped, dim=2, descending=True).values[:, :, :case["best"]].sum(2)
            kept = torch.sort(best, dim=1, descending=True, stable=True).indices[:, :case["kept"]]
            on = (kept.unsqueeze(2) == torch.arange(case["groups"], device=c.device)).any(1)
            c = torch.where(on.unsqueeze(2), grouped, -math.inf).view(c.shape)
        idx = torch.sort(c, dim=1, descending=True, stable=True).indices[:, :case["k"]]
        w = torch.gather(score, 1, idx).float()
        if case["normalize"]:
            w = w / w.sum(1, keepdim=True)
        return w * case["scale"], idx.to(torch.int32)
    t, n, m, r = (case[v] for v in ("T", "n", "N", "r"))
    index = s["index"].long()
    mine = (index.unsqueeze(1) == torch.arange(n, device=index.device)).float()
    # every row with every adapter, and of that the row's own
    inner = (s["x"].float() @ s["down"].float().transpose(0, 1).reshape(case["K"], n * r)).view(t, n, r)
    inner = inner * (mine * s["scale"]).unsqueeze(2)
    y = inner.reshape(t, n * r) @ s["up"].float().reshape(n * r, m)
    if case["base"]:
        y = y + s["base"].float()
    return y.to(_DT[case["out"]])


# ------------------------------------------------------------------------------------------------- interface


def prepare(case, seed):
    s = _inputs(case, seed)
    return _prepare_own(case, s) if own else (case, s)


def run(state):
    return state() if own else _plain(*state)


def work(case):
    op = case["op"]
    if op == "norm":
        t, h, size = case["T"], case["H"], _SIZE[case["dtype"]]
        scales = {"": 0, "tensor": 4, "row": 4 * t, "group": 4 * t * h // case["group"] if case["group"] else 0}[case["scales"]]
        return {"bytes": t * h * (size * (3 if case["residual"] else 1) + _SIZE[case["out"]]) + h * _SIZE[case["gamma"]] + scales,
                "flops": 6 * t * h}
    if op == "norm_grad":
        t, h, size = case["T"], case["H"], _SIZE[case["dtype"]]
        return {"bytes": t * h * size * (4 if case["residual"] else 3) + h * (_SIZE[case["gamma"]] + 4), "flops": 12 * t * h}
    if op == "route":
        t, e = case["T"], case["E"]
        return {"bytes": t * e * _SIZE[case["dtype"]] + 8 * t * case["k"] + (4 * e if case["bias"] else 0), "flops": 8 * t * e}
    t, n, k, m, r, size = case["T"], case["n"], case["K"], case["N"], case["r"], _SIZE[case["dtype"]]
    on = t * (1.0 - case["none"])
    used = n * (1.0 - (1.0 - 1.0 / n) ** on) if case["order"] == "mixed" else min(n, t)  # adapters that some row has, about
    return {"bytes": on * k * size + t * m * _SIZE[case["out"]] * (2 if case["base"] else 1) + used * (k + m) * r * size + 4 * t,
            "flops": 2 * on * r * (k + m)}


# ------------------------------------------------------------------------------------- the values in 64 bits


def exact(case, seed):
    s, op = _inputs(case, seed), case["op"]
    if op == "norm":
        h = s["x"].double()
        if case["residual"]:
            h = h + s["residual"].double()
        total = (h,) if case["residual"] else ()
        y = torch.nn.functional.normalize(h, dim=1, eps=0.0)  # h / |h|
        norm2 = h.square().sum(1, keepdim=True)
        y = y * torch.sqrt(norm2 / (norm2 / case["H"] + EPS)) * s["gamma"].double()
        if not case["scales"]:
            return (y,) + total
        limit = _LIMIT[case["out"]]
        if case["scales"] == "tensor":
            y, made = y / s["scale"].double(), ()
        else:
            width = case["group"] or case["H"]
            made = (torch.stack([p.abs().max(1).values for p in y.split(width, 1)], 1) / limit,)
            y = y / made[0].repeat_interleave(width, 1)
        # what 8 bits hold: whole numbers, or three binary digits behind the leading one and no exponent below -6
        if case["out"] == "s8":
            q = torch.round(y).clamp(-128, 127)
        else:
            step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
            q = (torch.round(y / step) * step).clamp(-limit, limit)
        return (q,) + made + total
    if op == "norm_grad":
        h = s["h"].double().requires_grad_()
        gamma = s["gamma"].double().requires_grad_()
        y = h / torch.sqrt(h.square().mean(1, keepdim=True) + EPS) * gamma
        dh, dgamma = torch.autograd.grad(y, (h, gamma), s["dy"].double())
        return dh + s["dsum"].double() if case["residual"] else dh, dgamma
    if op == "route":
        l = s["logits"].double()
        score = (torch.sigmoid(l) if case["scoring"] == "sigmoid" else torch.softmax(l, 1)).cpu().numpy()
        c = score + s["bias"].double().cpu().numpy() if case["bias"] else score.copy()
        t, e, groups = case["T"], case["E"], case["groups"]
        if groups > 1:
            rank = np.partition(c.reshape(t, groups, -1), -case["best"], 2)[:, :, -case["best"]:].sum(2)
            out = np.argsort(-rank, axis=1, kind="stable")[:, case["kept"]:]
            c.reshape(t, groups, -1)[np.arange(t)[:, None], out] = -np.inf
        idx = np.argsort(-c, axis=1, kind="stable")[:, :case["k"]]
        w = np.take_along_axis(score, idx, 1)
        if case["normalize"]:
            w = w / w.sum(1, keepdims=True)
        return torch.from_numpy(w * case["scale"]).cuda(), torch.from_numpy(idx.astype(np.int32)).cuda()
    y = s["base"].double() if case["base"] else torch.zeros((case["T"], case["N"]), dtype=torch.float64, device="cuda")
    for i in range(case["n"]):
        on = (s["index"] == i).nonzero()[:, 0]
        if on.numel():
            y[on] += s["scale"][i].double() * ((s["x"][on].double() @ s["down"][i].double()) @ s["up"][i].double())
    return y

"""Performance cases of the operators around a mixture-of-experts layer's products, and of dropout.

The experts' products themselves are ``dnnl::matmul`` on grouped memory (``perf/cases.py``).  These are the operators
that lead into them and out of them: the router's choice, the sort of the tokens into grouped rows, the weighted way
back with residual and dropout, dropout by itself, and the gradient of each.

``op`` of a case
  route          logits [T, E] -> the k experts of each token and their weights
  route_grad     gradient of the weights -> gradient of the logits
  dispatch       tokens [T, H] -> rows sorted by expert [T k, H], group offsets, the position of every slot
  dispatch_grad  gradient of the sorted rows -> gradient of the tokens (a sum over each token's rows)
  combine        the experts' rows back to tokens, weighted, + residual, dropout in between
  combine_grad   gradient of the tokens -> gradients of the rows and of the weights
  dropout        residual + dropout(x)
  dropout_grad   gradient of x, with the mask made again from the seed
"""
import math

import numpy as np
import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_CODE = {"f16": 1, "bf16": 2, "f32": 3, "s32": 4, "s64": 16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # token generation, one sequence: the router of a 64-expert layer (a few hundred bytes; latency)
        {"name": "route_token", "op": "route", "T": 1, "E": 64, "k": 8, "dtype": "f32", "scoring": "softmax",
         "normalize": True, "scale": 1.0},
        # a full batch of prompts, a wide 256-expert router with 16-bit logits, probabilities over all experts
        {"name": "route_prefill", "op": "route", "T": 8192, "E": 256, "k": 8, "dtype": "bf16", "scoring": "softmax",
         "normalize": False, "scale": 1.0},
        # training step of a router with sigmoid scores normalised over the chosen experts; an odd batch
        {"name": "route_grad", "op": "route_grad", "T": 8191, "E": 160, "k": 6, "dtype": "f32", "scoring": "sigmoid",
         "normalize": True, "scale": 2.5},
        # token generation on the 8 experts one GPU holds
        {"name": "dispatch_decode", "op": "dispatch", "T": 37, "E": 8, "k": 2, "H": 4096, "dtype": "bf16", "pad": 0.0,
         "pitch": 0},
        # a full batch of prompts over 64 experts: the largest of the forward cases
        {"name": "dispatch_prefill", "op": "dispatch", "T": 8192, "E": 64, "k": 8, "H": 4096, "dtype": "bf16",
         "pad": 0.0, "pitch": 0},
        # a ragged batch with padding tokens that go to no expert, an odd width, tokens inside a wider buffer
        {"name": "dispatch_ragged", "op": "dispatch", "T": 3001, "E": 160, "k": 6, "H": 2047, "dtype": "f16",
         "pad": 0.15, "pitch": 2053},
        # training: the gradient of the tokens is the sum over their rows' gradients
        {"name": "dispatch_grad", "op": "dispatch_grad", "T": 4096, "E": 64, "k": 8, "H": 4096, "dtype": "bf16",
         "pad": 0.0},
        # token generation, one sequence: eight experts' rows back into the residual stream
        {"name": "combine_token", "op": "combine", "T": 1, "E": 64, "k": 8, "H": 4096, "dtype": "bf16", "out": "bf16",
         "weights": True, "residual": True, "p": 0.0, "pad": 0.0, "pitch": 0},
        # training step, forward: a full batch back into the residual stream, with dropout
        {"name": "combine_train", "op": "combine", "T": 8192, "E": 64, "k": 8, "H": 4096, "dtype": "bf16", "out": "bf16",
         "weights": True, "residual": True, "p": 0.1, "pad": 0.0, "pitch": 0},
        # the same step backward: gradients of the rows and of the weights; some tokens are padding
        {"name": "combine_grad", "op": "combine_grad", "T": 4096, "E": 64, "k": 8, "H": 4096, "dtype": "bf16",
         "p": 0.1, "pad": 0.05, "pitch": 0},
        # dropout of a dense sublayer's output on the way into the residual stream
        {"name": "dropout_residual", "op": "dropout", "M": 8192, "N": 4096, "dtype": "bf16", "residual": True, "p": 0.1,
         "pitch": 0},
        # its gradient in 32 bits, an odd width inside a wider buffer
        {"name": "dropout_grad", "op": "dropout_grad", "M": 4099, "N": 1367, "dtype": "f32", "residual": False, "p": 0.25,
         "pitch": 1371},
    ]


def _log_int(rng, lo, hi):
    v = max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))
    return v + 1 if v % 1024 == 0 and v % 3 == 0 else v


def _width(rng):
    """Three of four hidden sizes are multiples of 64, as layers are; the others any number, odd ones among them."""
    h = _log_int(rng, 64, 8192)
    if rng.random() < 0.75:
        h = max(64, h // 64 * 64)
        h += 64 if h % 1024 == 0 and h % 3 == 0 else 0
    return h


def draw(rng):
    op = rng.choice(["route", "route_grad", "dispatch", "dispatch_grad", "combine", "combine_grad", "dropout",
                     "dropout_grad"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op.startswith("dropout"):
        m, n = _log_int(rng, 1, 16384), _width(rng)
        while m * n > 8192 * 4096:
            m //= 2
        return {"op": op, "M": m, "N": n, "dtype": dtype, "residual": op == "dropout" and rng.random() < 0.5,
                "p": rng.choice([0.05, 0.1, 0.2, 0.5]), "pitch": n + rng.randint(1, 64) if rng.random() < 0.25 else 0}
    t, e = _log_int(rng, 1, 8192), _log_int(rng, 4, 512)
    k = min(e, rng.choice([1, 2, 4, 6, 8]))
    c = {"op": op, "T": t, "E": e, "k": k, "dtype": dtype}
    if op.startswith("route"):
        c.update(scoring=rng.choice(["softmax", "sigmoid"]), normalize=rng.random() < 0.5, scale=rng.choice([1.0, 2.5]))
        return c
    h = _width(rng)
    while t * k * h * _SIZE[dtype] > 8192 * 8 * 4096 * 2:
        t = c["T"] = max(1, t // 2)
    c.update(H=h, pad=rng.choice([0.0, 0.0, 0.1, 0.4]))
    if op != "dispatch_grad":
        c["pitch"] = h + rng.randint(1, 64) if rng.random() < 0.25 else 0
    if op.startswith("combine"):
        c["p"] = rng.choice([0.0, 0.0, 0.1, 0.3])
    if op == "combine":
        c.update(out=rng.choice([dtype, "f32"]), weights=True, residual=rng.random() < 0.7)
    return c


# ---------------------------------------------------------------------------------------------------- inputs


def _logits(g, case):
    """A router's logits: unit normal, and experts that are more in demand than others."""
    t, e = case["T"], case["E"]
    demand = torch.randn(e, generator=g, device="cuda") * 0.5
    return (torch.randn((t, e), generator=g, device="cuda") + demand).to(_DT.get(case["dtype"], torch.float32))


def _choose(logits, k):
    """The k largest of each row, ties to the lowest index; masked (-inf, NaN) ones give index -1."""
    l = torch.where(torch.isnan(logits), -math.inf, logits.float())
    ids = torch.arange(l.shape[1], device=l.device)
    out = []
    for _ in range(k):
        top = l.amax(1, keepdim=True)
        i = torch.where(l == top, ids, l.shape[1]).amin(1, keepdim=True)
        out.append(torch.where(top == -math.inf, -1, i))
        l = torch.where(ids == i, -math.inf, l)
    return torch.cat(out, 1).to(torch.int32)


def _rows(g, shape, dtype, pitch=0, scale=1.0):
    """A matrix of unit normal values, with `pitch` elements from row to row where that is given."""
    m, n = shape
    t = (torch.randn((m, pitch or n), generator=g, device="cuda") * scale).to(_DT[dtype])
    return t[:, :n]


def _sorted_positions(indices, experts):
    """Offsets (cumulative ends) and the position of every slot in the stable order by expert."""
    flat = indices.reshape(-1).long()
    flat = torch.where((flat < 0) | (flat >= experts), experts, flat)  # slots without an expert go last
    expert, slot = torch.sort(flat, stable=True)
    ends = torch.searchsorted(expert, torch.arange(experts, device=flat.device), right=True)
    row = torch.arange(flat.numel(), device=flat.device)
    positions = torch.empty_like(flat)
    positions[slot] = torch.where(expert < experts, row, -1)
    return ends.to(torch.int32), positions.to(torch.int32).view(indices.shape)


def _inputs(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op, s = case["op"], {}
    if op.startswith("dropout"):
        s["x"] = _rows(g, (case["M"], case["N"]), case["dtype"], case["pitch"])
        if case["residual"]:
            s["residual"] = _rows(g, (case["M"], case["N"]), case["dtype"])
        s["seed"] = torch.randint(0, 2 ** 62, (2,), generator=g, device="cuda", dtype=torch.int64)
        return s
    if op.startswith("route"):
        s["logits"] = _logits(g, case)
        if op == "route_grad":
            s["indices"] = _choose(s["logits"], case["k"])
            s["dweights"] = torch.randn((case["T"], case["k"]), generator=g, device="cuda")
        return s
    t, k, h = case["T"], case["k"], case["H"]
    logits = _logits(g, {"T": t, "E": case["E"], "dtype": "f32"})
    indices = _choose(logits, k)
    weights = torch.softmax(torch.gather(logits, 1, indices.long()), 1).contiguous()
    padding = torch.rand((t, 1), generator=g, device="cuda") < case["pad"]
    indices = torch.where(padding, -1, indices).contiguous()
    if op == "dispatch":
        s["x"], s["indices"] = _rows(g, (t, h), case["dtype"], case["pitch"]), indices
        return s
    s["offsets"], s["positions"] = _sorted_positions(indices, case["E"])
    s["rows"] = _rows(g, (t * k, h), case["dtype"])
    if op == "combine":
        s["weights"] = weights
        if case["residual"]:
            s["residual"] = _rows(g, (t, h), case["out"], case["pitch"])
    if op == "combine_grad":
        s["weights"] = weights
        s["dy"] = _rows(g, (t, h), case["dtype"], case["pitch"])
    if case.get("p"):
        s["seed"] = torch.randint(0, 2 ** 62, (2,), generator=g, device="cuda", dtype=torch.int64)
    return s


# ------------------------------------------------------------------------------- the framework's operators


class _Call:
    """One primitive with the memory objects that wrap the program's device buffers."""

    def __init__(self):
        from onednn_b200 import api
        self.api = api
        self.eng = api.engine(api.engine.kind.gpu, torch.cuda.current_device())
        self.strm = api.stream(self.eng, torch.cuda.current_stream().cuda_stream)
        self.args, self.keep = {}, []

    def bind(self, arg, t):
        names = {torch.float32: "f32", torch.bfloat16: "bf16", torch.float16: "f16", torch.int32: "s32",
                 torch.int64: "s64"}
        md = self.api.memory.desc(t.shape, _CODE[names[t.dtype]], tuple(t.stride()))
        self.args[arg] = self.api.memory(md, self.eng, t.data_ptr())
        self.keep.append(t)
        return md

    def bind_grouped(self, arg, t, offsets):
        names = {torch.float32: "f32", torch.bfloat16: "bf16", torch.float16: "f16"}
        md = self.api.memory.desc.grouped(t.shape, _CODE[names[t.dtype]], 0, offsets.numel())
        self.args[arg] = self.api.memory(md, self.eng, handles=[t.data_ptr(), offsets.data_ptr()])
        self.keep += [t, offsets]
        return md

    def make(self, primitive, pd, outputs):
        self.prim, self.outputs = primitive(pd), outputs
        return self

    def __call__(self):
        self.prim.execute(self.strm, self.args)
        return self.outputs


def _empty(shape, dtype):
    return torch.empty(shape, device="cuda", dtype=dtype)


def _prepare_own(case, s):
    c = _Call()
    api, op = c.api, case["op"]
    if op.startswith("route"):
        mode = dict(scoring=getattr(api.scoring, case["scoring"]), normalize=case["normalize"], scale=case["scale"])
        logits = c.bind(api.ARG_SRC, s["logits"])
        if op == "route":
            w, i = _empty((case["T"], case["k"]), torch.float32), _empty((case["T"], case["k"]), torch.int32)
            pd = api.moe_route.primitive_desc(c.eng, logits, c.bind(api.ARG_DST, w), c.bind(api.ARG_DST_1, i), **mode)
            return c.make(api.moe_route, pd, (w, i))
        d = torch.empty_like(s["logits"])
        pd = api.moe_route_backward.primitive_desc(
            c.eng, logits, c.bind(api.ARG_SRC_1, s["indices"]), c.bind(api.ARG_DIFF_DST, s["dweights"]),
            c.bind(api.ARG_DIFF_SRC, d), **mode)
        return c.make(api.moe_route_backward, pd, d)
    if op.startswith("dropout"):
        y = _empty((case["M"], case["N"]), _DT[case["dtype"]])
        residual = c.bind(api.ARG_SRC_2, s["residual"]) if case["residual"] else None
        c.bind(api.ARG_ATTR_DROPOUT_SEED, s["seed"])
        pd = api.dropout.primitive_desc(c.eng, c.bind(api.ARG_SRC, s["x"]), c.bind(api.ARG_DST, y), case["p"],
                                        residual_md=residual)
        return c.make(api.dropout, pd, y)
    t, k, h = case["T"], case["k"], case["H"]
    if op == "dispatch":
        rows = _empty((t * k, h), _DT[case["dtype"]])
        offsets, pos = _empty((case["E"],), torch.int32), _empty((t, k), torch.int32)
        pd = api.moe_dispatch.primitive_desc(c.eng, c.bind(api.ARG_SRC, s["x"]), c.bind(api.ARG_SRC_1, s["indices"]),
                                             c.bind_grouped(api.ARG_DST, rows, offsets), c.bind(api.ARG_DST_1, pos))
        return c.make(api.moe_dispatch, pd, (rows, offsets, pos))
    pos = c.bind(api.ARG_SRC_1, s["positions"])
    src = c.bind_grouped(api.ARG_SRC, s["rows"], s["offsets"])
    weights = c.bind(api.ARG_WEIGHTS, s["weights"]) if "weights" in s else None
    if "seed" in s:
        c.bind(api.ARG_ATTR_DROPOUT_SEED, s["seed"])
    if op == "combine_grad":
        drows, dw = torch.empty_like(s["rows"]), torch.empty_like(s["weights"])
        pd = api.moe_combine_backward.primitive_desc(
            c.eng, c.bind(api.ARG_DIFF_DST, s["dy"]), src, pos, weights,
            c.bind_grouped(api.ARG_DIFF_SRC, drows, s["offsets"]), c.bind(api.ARG_DIFF_WEIGHTS, dw), dropout_p=case["p"])
        return c.make(api.moe_combine_backward, pd, (drows, dw))
    y = _empty((t, h), _DT[case.get("out", case["dtype"])])
    residual = c.bind(api.ARG_SRC_2, s["residual"]) if "residual" in s else None
    pd = api.moe_combine.primitive_desc(c.eng, src, pos, c.bind(api.ARG_DST, y), weights_md=weights,
                                        residual_md=residual, dropout_p=case.get("p", 0.0))
    return c.make(api.moe_combine, pd, y)


# ------------------------------------------------------------------------------------------- plain forms


def _philox(seed, count):
    """`count` 32-bit words (as int64): word i is word i % 4 of Philox4x32 with ten rounds (Salmon, Moraes, Dror, Shaw:
    Parallel random numbers: as easy as 1, 2, 3; 2011), counter (i / 4, offset), key seed; seed = (seed, offset)."""
    mask = 0xffffffff
    i = torch.arange((count + 3) // 4, device=seed.device, dtype=torch.int64)
    key = [seed[0] & mask, (seed[0] >> 32) & mask]
    c = [i & mask, i >> 32, (seed[1] & mask).expand_as(i), ((seed[1] >> 32) & mask).expand_as(i)]

    def product(a, b):  # the two words of a 64-bit product
        high = (a * (b >> 16) + ((a * (b & 0xffff)) >> 16)) >> 16
        return high, (a * b) & mask

    for r in range(10):
        h0, l0 = product(0xD2511F53, c[0])
        h1, l1 = product(0xCD9E8D57, c[2])
        c = [h1 ^ c[1] ^ key[0], l1, h0 ^ c[3] ^ key[1], l0]
        key = [(key[0] + 0x9E3779B9) & mask, (key[1] + 0xBB67AE85) & mask]
    return torch.stack(c, 1).view(-1)[:count]


def _dropout(x, seed, p):
    p = float(np.float32(p))  # the probability is given in 32 bits
    keep = _philox(seed, x.numel()).view(x.shape) >= int(p * 2 ** 32)
    return torch.where(keep, x * (1.0 / (1.0 - p)), 0.0)


def _plain(case, s):
    op = case["op"]
    if op == "route":
        l = s["logits"].float()
        idx = _choose(l, case["k"])
        v = torch.gather(l, 1, idx.clamp_min(0).long())
        v = torch.where(idx < 0, -math.inf, v)
        if case["scoring"] == "sigmoid":
            w = 1.0 / (1.0 + torch.exp(-v))
            if case["normalize"]:
                w = w / w.sum(1, keepdim=True)
        else:
            w = torch.exp(v - v[:, :1])
            total = w if case["normalize"] else torch.exp(l - v[:, :1])
            w = w / total.sum(1, keepdim=True)
        return w * case["scale"], idx
    if op == "route_grad":
        l, idx, c = s["logits"].float(), s["indices"], case["scale"]
        hot = idx.unsqueeze(2) == torch.arange(case["E"], device=l.device)
        g = torch.where(hot, s["dweights"].unsqueeze(2), 0.0).sum(1) * c
        chosen = hot.any(1)
        if case["scoring"] == "sigmoid":
            p = 1.0 / (1.0 + torch.exp(-l))
            slope = torch.where(chosen, p * (1.0 - p), 0.0)
            if case["normalize"]:
                total = torch.where(chosen, p, 0.0).sum(1, keepdim=True)
                d = slope / total * (g - (g * p).sum(1, keepdim=True) / total)
            else:
                d = slope * g
        else:
            e = torch.exp(l - l.amax(1, keepdim=True))
            if case["normalize"]:
                e = torch.where(chosen, e, 0.0)
            p = e / e.sum(1, keepdim=True)
            d = p * (g - (g * p).sum(1, keepdim=True))
        return d.to(s["logits"].dtype)
    if op.startswith("dropout"):
        y = _dropout(s["x"].float(), s["seed"], case["p"])
        if case["residual"]:
            y = y + s["residual"].float()
        return y.to(s["x"].dtype)
    t, k, h = case["T"], case["k"], case["H"]
    if op == "dispatch":
        offsets, pos = _sorted_positions(s["indices"], case["E"])
        flat = pos.view(-1).long()
        kept = flat >= 0
        rows = torch.zeros((t * k, h), device="cuda", dtype=_DT[case["dtype"]])
        token = torch.arange(t * k, device="cuda") // k
        rows[flat[kept]] = s["x"][token[kept]]
        return rows, offsets, pos
    pos = s["positions"].long()
    kept = (pos >= 0).unsqueeze(2)
    rows = torch.where(kept, s["rows"][pos.clamp_min(0)].float(), 0.0)
    if op == "combine_grad":
        dy = s["dy"].float()
        if case["p"]:
            dy = _dropout(dy, s["seed"], case["p"])
        dw = (rows * dy.unsqueeze(1)).sum(2)
        d = s["weights"].unsqueeze(2) * dy.unsqueeze(1)
        drows = torch.zeros((t * k, h), device="cuda", dtype=s["rows"].dtype)
        where = pos.view(-1)
        drows[where[where >= 0]] = d.view(t * k, h)[where >= 0].to(s["rows"].dtype)
        return drows, dw
    if op == "combine":
        rows = rows * s["weights"].unsqueeze(2)
    y = rows.sum(1)
    if case.get("p"):
        y = _dropout(y, s["seed"], case["p"])
    if "residual" in s:
        y = y + s["residual"].float()
    return y.to(_DT[case.get("out", case["dtype"])])


# ------------------------------------------------------------------------------------------------- interface


def prepare(case, seed):
    s = _inputs(case, seed)
    return _prepare_own(case, s) if own else (case, s)


def run(state):
    return state() if own else _plain(*state)


def work(case):
    op = case["op"]
    if op.startswith("dropout"):
        n = case["M"] * case["N"]
        return {"bytes": n * _SIZE[case["dtype"]] * (3 if case["residual"] else 2) + 16, "flops": 2 * n}
    t, k, e, size = case["T"], case["k"], case["E"], _SIZE[case["dtype"]]
    if op == "route":
        return {"bytes": t * e * size + 8 * t * k, "flops": 4 * t * e}
    if op == "route_grad":
        return {"bytes": 2 * t * e * size + 8 * t * k, "flops": 6 * t * e}
    h = case["H"]
    if op == "dispatch":
        return {"bytes": (t + t * k) * h * size + 8 * t * k + 4 * e, "flops": t * k}
    if op == "dispatch_grad":
        return {"bytes": (t + t * k) * h * size + 4 * t * k, "flops": t * k * h}
    if op == "combine":
        out = _SIZE[case["out"]] * (2 if case["residual"] else 1)
        return {"bytes": t * k * h * size + t * h * out + 8 * t * k, "flops": 2 * t * k * h}
    return {"bytes": (t + 2 * t * k) * h * size + 12 * t * k, "flops": 3 * t * k * h}


# ------------------------------------------------------------------------------------- the values in 64 bits


def _exact_keep(seed, m, n, p):
    """1 / (1 - p) where an element is kept and 0 where it is dropped, by the same generator in numpy's integers."""
    p = float(np.float32(p))
    seed, offset = (int(v) for v in seed.cpu())
    word = np.uint64(0xffffffff)
    i = np.arange((m * n + 3) // 4, dtype=np.uint64)
    x0, x1 = i & word, i >> np.uint64(32)
    x2 = np.full_like(i, offset & 0xffffffff)
    x3 = np.full_like(i, offset >> 32 & 0xffffffff)
    k0, k1 = seed & 0xffffffff, seed >> 32 & 0xffffffff
    for _ in range(10):
        a, b = x0 * np.uint64(0xD2511F53), x2 * np.uint64(0xCD9E8D57)
        x0 = (b >> np.uint64(32)) ^ x1 ^ np.uint64(k0)
        x2 = (a >> np.uint64(32)) ^ x3 ^ np.uint64(k1)
        x1, x3 = b & word, a & word
        k0, k1 = k0 + 0x9E3779B9 & 0xffffffff, k1 + 0xBB67AE85 & 0xffffffff
    u = np.empty((i.size, 4), np.uint64)
    u[:, 0], u[:, 1], u[:, 2], u[:, 3] = x0, x1, x2, x3
    keep = torch.from_numpy((u.reshape(-1)[:m * n] >= np.uint64(int(p * 2.0 ** 32))).reshape(m, n)).cuda()
    return keep.double() / (1.0 - p)


def exact(case, seed):
    s, op = _inputs(case, seed), case["op"]
    if op.startswith("dropout"):
        y = s["x"].double() * _exact_keep(s["seed"], case["M"], case["N"], case["p"])
        return y + s["residual"].double() if case["residual"] else y
    t, k = case["T"], case["k"]
    if op.startswith("route"):
        z = s["logits"].double().requires_grad_(op == "route_grad")
        if op == "route":
            idx = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :k]
        else:
            idx = s["indices"].long()
        score = torch.softmax(z, 1) if case["scoring"] == "softmax" else torch.sigmoid(z)
        w = torch.gather(score, 1, idx)
        if case["normalize"]:
            w = w / w.sum(1, keepdim=True)
        w = w * case["scale"]
        if op == "route":
            return w, idx.to(torch.int32)
        return torch.autograd.grad(w, z, s["dweights"].double())[0]
    h = case["H"]
    if op == "dispatch":
        flat = s["indices"].view(-1).cpu().numpy()
        flat = np.where((flat < 0) | (flat >= case["E"]), case["E"], flat)
        order = np.argsort(flat, kind="stable")
        kept = int((flat < case["E"]).sum())
        pos = np.full(t * k, -1, np.int32)
        pos[order[:kept]] = np.arange(kept)
        ends = np.cumsum(np.bincount(flat, minlength=case["E"] + 1)[:case["E"]]).astype(np.int32)
        rows = torch.zeros((t * k, h), dtype=torch.float64, device="cuda")
        rows[:kept] = s["x"].double()[torch.from_numpy(order[:kept] // k).cuda()]
        return rows, torch.from_numpy(ends).cuda(), torch.from_numpy(pos.reshape(t, k)).cuda()
    pos = s["positions"].long()
    if op == "combine_grad":
        dy = s["dy"].double()
        if case["p"]:
            dy = dy * _exact_keep(s["seed"], t, h, case["p"])
        drows = torch.zeros((t * k, h), dtype=torch.float64, device="cuda")
        dw = torch.zeros((t, k), dtype=torch.float64, device="cuda")
        for j in range(k):
            on = pos[:, j] >= 0
            at = pos[on, j]
            drows[at] = s["weights"][on, j:j + 1].double() * dy[on]
            dw[on, j] = (s["rows"][at].double() * dy[on]).sum(1)
        return drows, dw
    y = torch.zeros((t, h), dtype=torch.float64, device="cuda")
    for j in range(k):
        on = pos[:, j] >= 0
        r = s["rows"][pos[on, j]].double()
        y[on] += r * s["weights"][on, j:j + 1].double() if op == "combine" else r
    if case.get("p"):
        y = y * _exact_keep(s["seed"], t, h, case["p"])
    return y + s["residual"].double() if "residual" in s else y

"""Plain 64-bit forms of the operators around an expert layer's products and of dropout, and the calls through the
library that the tests compare with them (torch tensors on the device behind memory objects)."""
import numpy as np

U32 = np.uint64(0xffffffff)
EPS = 2.0 ** -24  # unit roundoff of 32-bit floats


def philox_blocks(seed, offset, block):
    """the four words of each block of Philox4x32-10: counter (block, offset), key seed"""
    c = [block & U32, block >> np.uint64(32), np.full_like(block, offset & 0xffffffff),
         np.full_like(block, offset >> 32 & 0xffffffff)]
    k = [seed & 0xffffffff, seed >> 32 & 0xffffffff]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & U32, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & U32]
        k = [k[0] + 0x9E3779B9 & 0xffffffff, k[1] + 0xBB67AE85 & 0xffffffff]
    return np.stack(c, 1)


def philox_words(seed, offset, first, count):
    """Words first .. first + count: word i is word i % 4 of block i / 4."""
    b0 = first // 4
    words = philox_blocks(seed, offset, np.arange(b0, (first + count + 3) // 4, dtype=np.uint64)).reshape(-1)
    return words[first - 4 * b0:first - 4 * b0 + count]


def keep_mask(shape, p, seed, offset):
    """kept elements, and 1 / (1 - p) with p as the 32-bit number it is"""
    p = float(np.float32(p))
    n = int(np.prod(shape))
    return (philox_words(seed, offset, 0, n) >= np.uint64(int(p * 2.0 ** 32))).reshape(shape), (1 / (1 - p) if p < 1 else 0.0)


def dropout(x, p, seed, offset):
    keep, scale = keep_mask(x.shape, p, seed, offset)
    return np.where(keep, x * scale, 0.0)


def choose(logits, k):
    """indices of the k largest of each row, ties to the lowest index; -1 where only masked logits are left"""
    l = np.where(np.isnan(logits), -np.inf, logits)
    idx = np.argsort(-l, axis=1, kind="stable")[:, :k]
    return np.where(np.take_along_axis(l, idx, 1) > -np.inf, idx, -1).astype(np.int32)


def route_weights(logits, idx, scoring, normalize, scale):
    """weights of the given choices, differentiable by differences: the choice is fixed"""
    l = np.where(np.isnan(logits), -np.inf, logits)
    with np.errstate(all="ignore"):
        v = np.where(idx >= 0, np.take_along_axis(l, np.maximum(idx, 0), 1), -np.inf)
        if scoring == "softmax":
            over = v if normalize else l
            m = np.maximum(np.max(l, 1, keepdims=True), -1e300)
            w = np.exp(v - m) / np.exp(over - m).sum(1, keepdims=True)
        else:
            ls = -np.logaddexp(0.0, -v)
            if normalize:
                m = np.maximum(np.max(ls, 1, keepdims=True), -1e300)
                w = np.exp(ls - m)
                w = w / w.sum(1, keepdims=True)
            else:
                w = np.exp(ls)
    return np.where(idx >= 0, w, 0.0) * scale


def route_backward(logits, idx, g, scoring, normalize, scale):
    """gradient of the logits, and the sum of the magnitudes that it is the difference of"""
    T, E = logits.shape
    l = np.where(np.isnan(logits), -np.inf, logits)
    d, size = np.zeros((T, E)), np.zeros((T, E))
    w = route_weights(logits, idx, scoring, normalize, 1.0)
    g = np.where(idx >= 0, g * scale, 0.0)
    inner, inner_size = (g * w).sum(1), (np.abs(g) * w).sum(1)
    for t in range(T):
        if scoring == "softmax" and not normalize and np.isfinite(l[t]).any():
            p = np.exp(l[t] - l[t].max())
            p /= p.sum()
            d[t] -= p * inner[t]
            size[t] += p * inner_size[t]
        for j in range(idx.shape[1]):
            i = idx[t, j]
            if i < 0:
                continue
            if scoring == "softmax":
                d[t, i] += w[t, j] * (g[t, j] - (inner[t] if normalize else 0))
                size[t, i] += w[t, j] * (abs(g[t, j]) + (inner_size[t] if normalize else 0))
            else:
                slope = 1 / (1 + np.exp(l[t, i]))  # 1 - s
                d[t, i] += w[t, j] * slope * (g[t, j] - (inner[t] if normalize else 0))
                size[t, i] += w[t, j] * slope * (abs(g[t, j]) + (inner_size[t] if normalize else 0))
    return d, size


def sort_slots(indices, experts):
    """(offsets, positions) of the stable sort by expert; the slots in row order"""
    flat = indices.reshape(-1).astype(np.int64)
    flat = np.where((flat < 0) | (flat >= experts), experts, flat)
    order = np.argsort(flat, kind="stable")
    order = order[:int((flat < experts).sum())]
    pos = np.full(flat.size, -1, np.int32)
    pos[order] = np.arange(order.size)
    ends = np.cumsum(np.bincount(flat, minlength=experts + 1)[:experts]).astype(np.int32)
    return ends, pos.reshape(indices.shape), order


def out_slack(value, dtype):
    """half a unit in the last place of a value stored in dtype (bits of the significand, exponent of the least normal);
    a value that falls just short of a power of two may be rounded with the unit above it"""
    bits, least = {"f32": (24, -126), "bf16": (8, -126), "f16": (11, -14)}[dtype]
    exponent = np.floor(np.log2(np.maximum(np.abs(value) * (1 + 2.0 ** -bits), 2.0 ** least)))
    return 2.0 ** (exponent - bits) * (1 + 1e-9)


class Call:
    """One primitive and its memory objects on the library's own stream or a caller's."""

    CODE = {"f16": 1, "bf16": 2, "f32": 3, "s32": 4, "s8": 5, "u8": 6, "s64": 16}

    def __init__(self, eng, cuda_stream=None):
        import torch
        from onednn_b200 import api
        self.torch, self.api, self.eng = torch, api, eng
        self.strm = api.stream(eng, cuda_stream if cuda_stream is not None else torch.cuda.current_stream().cuda_stream)
        self.args, self.keep = {}, []

    def name(self, t):
        T = self.torch
        return {T.float32: "f32", T.bfloat16: "bf16", T.float16: "f16", T.int32: "s32", T.int64: "s64", T.int8: "s8",
                T.uint8: "u8"}[t.dtype]

    def bind(self, arg, t, open_dims=()):
        if t is None:
            return None
        api, code = self.api, self.CODE[self.name(t)]
        self.args[arg] = api.memory(api.memory.desc(tuple(t.shape), code, tuple(t.stride())), self.eng, t.data_ptr())
        self.keep.append(t)
        dims = [api.RUNTIME_DIM_VAL if d in open_dims else n for d, n in enumerate(t.shape)]
        strides = [api.RUNTIME_DIM_VAL if open_dims and d == 0 else n for d, n in enumerate(t.stride())]
        return api.memory.desc(dims, code, tuple(strides))

    def grouped(self, arg, t, offsets, open_rows=False):
        api, code = self.api, self.CODE[self.name(t)]
        md = api.memory.desc.grouped(tuple(t.shape), code, 0, offsets.numel())
        self.args[arg] = api.memory(md, self.eng, handles=[t.data_ptr(), offsets.data_ptr()])
        self.keep += [t, offsets]
        return api.memory.desc.grouped((api.RUNTIME_DIM_VAL, t.shape[1]), code, 0, offsets.numel()) if open_rows else md

    def run(self, primitive, pd):
        self.prim = primitive(pd)
        self.prim.execute(self.strm, self.args)
        return self


def torch_dtype(name):
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "s8": torch.int8, "s32": torch.int32}[name]


def device_matrix(a, dtype, pitch=0, offset=0):
    """a numpy matrix on the device in `dtype`, `pitch` elements from row to row, `offset` elements into its buffer"""
    import torch
    m, n = a.shape
    ld = pitch or n
    buf = torch.zeros(max(1, offset + m * ld), dtype=torch_dtype(dtype), device="cuda:0")
    t = buf[offset:offset + m * ld].view(m, ld)[:, :n]
    t.copy_(torch.from_numpy(np.ascontiguousarray(a)))
    return t


def host(t):
    return t.double().cpu().numpy() if t.dtype.is_floating_point else t.cpu().numpy()

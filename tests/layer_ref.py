"""Plain 64-bit forms of the norm in front of a quantized product and of the router with a bias and groups, with the bounds of
what 32-bit sums may be off, and the binding of 8-bit tensors that the tests use."""
import numpy as np

import token_ref as R

EPS = R.EPS
E4M3 = 10
LIMIT = {"s8": 127.0, "e4m3": 448.0}


class Call(R.Call):
    """also binds e4m3 tensors (torch.float8_e4m3fn)"""

    CODE = dict(R.Call.CODE, e4m3=E4M3)

    def name(self, t):
        return "e4m3" if t.dtype == self.torch.float8_e4m3fn else super().name(t)


def torch_dtype(name):
    import torch
    return torch.float8_e4m3fn if name == "e4m3" else R.torch_dtype(name)


def rounded(a, dtype):
    """64-bit numbers as `dtype` holds them"""
    import torch
    t = torch.from_numpy(np.ascontiguousarray(a))
    return t.to(torch_dtype(dtype)).double().numpy()


def norm(x, epsilon, weights=None, residual=None):
    """(y, the sum)"""
    h = x if residual is None else x + residual
    y = h / np.sqrt((h * h).mean(1, keepdims=True) + epsilon)
    return (y if weights is None else y * weights), h


# Relative error of y before it is rounded to its type, in units of 2^-24, an upper bound: the sum (1), squares added by a thread (at
# most 32 of them, in two sums or one), a warp (5) and a CTA (4), each square off by that of the sum twice (2): 43; the mean, epsilon
# and, at half of all that, the root: 24; its inverse (1) and two products (2).
NORM_UNITS = 28


def norm_backward(h, dy, epsilon, weights=None, dsum=None):
    """(gradient of the sum, of the weights), and for each the size of the terms that it is the difference of"""
    z = dy if weights is None else dy * weights
    r = 1 / np.sqrt((h * h).mean(1, keepdims=True) + epsilon)
    dh = r * z - h * r ** 3 * (h * z).mean(1, keepdims=True)
    size = r * np.abs(z) + np.abs(h) * r ** 3 * np.abs(h * z).mean(1, keepdims=True)
    if dsum is not None:
        dh, size = dh + dsum, size + np.abs(dsum)
    return dh, (dy * h * r).sum(0), size, np.abs(dy * h * r).sum(0)


# Error of the gradient of the sum over that size: r (25) three times, the sum of h z (43), and six roundings of the rest.
NORM_GRAD_UNITS = 125


def step_e4m3(v):
    """distance of the e4m3 values around |v|"""
    return 2.0 ** (np.floor(np.log2(np.maximum(np.abs(v), 2.0 ** -6))) - 3)


def check_8bit(q, v, units, out):
    """q (what the device stored) is `v` rounded to nearest and saturated, v off by `units` 2^-24 of itself before that"""
    limit, least = LIMIT[out], -128.0 if out == "s8" else -448.0
    off = units * EPS * np.abs(v)
    v = np.clip(v, least, limit)
    half = 0.5 if out == "s8" else step_e4m3(np.abs(v) + off) / 2
    assert (np.abs(q - v) <= half * (1 + 1e-12) + off).all(), np.abs(q - v).max()


def quantized(y, out, group):
    """(y / scale, scale) with the scale made per row (group 0) or per group of columns"""
    T, H = y.shape
    parts = y.reshape(T, -1, group or H)
    scale = np.abs(parts).max(2) / LIMIT[out]
    return (parts / scale[:, :, None]).reshape(T, H), scale


def choose(logits, bias, scoring, k, groups=1, kept=1, best=1):
    """indices of the k largest of score + bias in the kept groups of each row, ties to the lowest index; -1 where nothing is left"""
    T, E = logits.shape
    l = np.where(np.isnan(logits), -np.inf, logits)
    there = l > -np.inf
    with np.errstate(all="ignore"):
        if scoring == "sigmoid":
            s = 1 / (1 + np.exp(-l))
        else:
            e = np.exp(l - l.max(1, keepdims=True))
            s = e / e.sum(1, keepdims=True)
    b = np.zeros(E) if bias is None else bias
    c = np.where(there & (b > -np.inf), s + np.minimum(b, np.finfo(np.float32).max), -np.inf)
    if kept < groups:
        top = np.sort(c.reshape(T, groups, E // groups), axis=2)[:, :, ::-1][:, :, :best]
        rank = np.where(top[:, :, 0] > -np.inf, np.where(top > -np.inf, top, 0).sum(2), -np.inf)
        out = np.argsort(-rank, axis=1, kind="stable")[:, kept:]
        c.reshape(T, groups, E // groups)[np.arange(T)[:, None], out] = -np.inf
    idx = np.argsort(-c, axis=1, kind="stable")[:, :k]
    return np.where(np.take_along_axis(c, idx, 1) > -np.inf, idx, -1).astype(np.int32)


def low_rank(x, index, down, up, scale=None, base=None):
    """(base + scale[i] (x down[i]) up[i], terms of the second product, of both): the latter are sums of magnitudes"""
    T, N = x.shape[0], up.shape[2]
    y = np.zeros((T, N)) if base is None else base.copy()
    second, both = np.zeros((T, N)), np.zeros((T, N))
    for i in np.unique(index):
        if not 0 <= i < down.shape[0]:
            continue
        on, s = index == i, 1.0 if scale is None else scale[i]
        v = x[on] @ down[i]
        y[on] += s * (v @ up[i])
        second[on] = abs(s) * (np.abs(v) @ np.abs(up[i]))
        both[on] = abs(s) * ((np.abs(x[on]) @ np.abs(down[i])) @ np.abs(up[i]))
    return y, second, both


def low_rank_bound(y, second, both, base, K, r, dtype, out):
    """What the adapters' result may be off.  An MMA adds sixteen products to a sum; its sum may be cut instead of rounded: 2^-23
    of its terms' magnitudes each.  First product: at most K / 16 MMAs a warp, sums over 8 warps and 8 CTAs (16 roundings), the
    scale (2).  What 16-bit parts leave out: 2^-18 (two of bf16), 2^-27 (three), 2^-22 (two of f16, whose smallest parts are
    further down).  Second product: r / 16 MMAs a part on top of the base.  Then the output's rounding."""
    parts = 2.0 ** -22 if dtype == "f16" else 2.0 ** -27 if out == "f32" else 2.0 ** -18
    mmas = 3 * (r / 16 + 1) + 1
    b = 0 if base is None else np.abs(base)
    return both * (K / 16 + 20) * 2 * EPS + second * parts * (1 + 2.0 ** -8) + mmas * 2 * EPS * (second * 1.01 + b) + R.out_slack(y, out)

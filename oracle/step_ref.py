"""Float64 restatement of the operators around a training step's products: the norm of query and key
heads with their rotation, the norm of a gradient, AdamW (oracle; test infrastructure).

As in train_ref, a result comes with the sum of the absolute values of the terms it is made of: the
scale that the kernels' rounding errors are proportional to.
"""
from __future__ import annotations

import math

import numpy as np
import torch

from .train_ref import philox_words

Tensor = torch.Tensor


def head_norm_rope(x, w, cos, sin, eps, pos, dout=None):
    """x [B,S,H,D] (CPU, any dtype), w [D], cos / sin [rows, D], pos [B,S] table rows: {name: (value, scale)}
    for out and, with dout, dx and dw."""
    x, w, cos, sin = (t.double() for t in (x, w, cos, sin))
    D = x.shape[-1]
    h = D // 2
    c, s = cos[pos][:, :, None], sin[pos][:, :, None]
    r = (x.pow(2).sum(-1, keepdim=True) / D + eps).rsqrt()
    y = x * r * w
    out, mag = torch.empty_like(y), torch.empty_like(y)
    out[..., :h] = y[..., :h] * c[..., :h] - y[..., h:] * s[..., :h]
    out[..., h:] = y[..., h:] * c[..., h:] + y[..., :h] * s[..., h:]
    mag[..., :h] = (y[..., :h] * c[..., :h]).abs() + (y[..., h:] * s[..., :h]).abs()
    mag[..., h:] = (y[..., h:] * c[..., h:]).abs() + (y[..., :h] * s[..., h:]).abs()
    res = {"out": (out, mag)}
    if dout is None:
        return res
    g = dout.double()
    a, b = g[..., :h], g[..., h:]
    dy = torch.cat((a * c[..., :h] + b * s[..., h:], b * c[..., h:] - a * s[..., :h]), -1)
    ady = torch.cat(((a * c[..., :h]).abs() + (b * s[..., h:]).abs(), (b * c[..., h:]).abs() + (a * s[..., :h]).abs()), -1)
    xn = x * r
    u, au = dy * w, ady * w.abs()
    res["dx"] = (r * (u - xn * (u * xn).mean(-1, keepdim=True)),
                 r * (au + xn.abs() * (au * xn.abs()).mean(-1, keepdim=True)))
    res["dw"] = ((dy * xn).sum((0, 1, 2)), (ady * xn.abs()).sum((0, 1, 2)))
    return res


# ------------------------------------------------------------------------------------------ AdamW
SITE = 2 ** 32 - 1
FIRST, SECOND = (7, 7), (15, 14)  # bias of the exponent, exponent of a block's largest value


def decode(codes, scales, kind):
    """float32 [n] of uint8 codes [n] in blocks of 256 with their scales."""
    bias, top = kind
    code = codes.reshape(-1, 256).astype(np.int64)
    mag = code & 127 if kind == FIRST else code
    e, f = mag >> 3, (mag & 7).astype(np.float64)
    v = np.where(e > 0, np.ldexp(8 + f, e - 3 - bias), np.ldexp(f, -2 - bias))
    v = np.where((kind == FIRST) & (code > 127), -v, v)
    s = scales.astype(np.int64)[:, None]
    return np.where(s == 255, np.nan, np.ldexp(v, np.maximum(s, 32) - 127 - top)).astype(np.float32).reshape(-1)


def encode(x, words, kind):
    """(codes, scales) of float32 x [n]: rounded down, and up by a step where the part cut off and word / 2^16
    come to a step.  In exact arithmetic."""
    bias, top = kind
    x = x.reshape(-1, 256).astype(np.float64)
    big = np.abs(x).max(1)
    bad = ~np.isfinite(x).all(1)
    e = np.where(big > 0, np.frexp(np.where(bad, 1.0, np.maximum(big, 1e-300)))[1] - 1 + 127, 0)
    e = np.clip(e, 32, 254)
    y = np.ldexp(np.abs(np.where(bad[:, None], 0.0, x)), (127 + top - e)[:, None])
    lowest = 1 - bias
    ex = np.maximum(np.frexp(y)[1] - 1, lowest)
    n = np.floor(np.ldexp(y, 3 - ex) + words.reshape(-1, 256) / 65536.0).astype(np.int64)
    # n steps of 2^(ex - 3): 8 and more is a normal number, 16 the next binade's first.
    code = np.where(n >= 8, ((ex + bias) << 3) + (n - 8), n)
    if kind == FIRST:
        code = code | (np.signbit(x) << 7)
    else:
        code = np.maximum(code, (x > 0).astype(np.int64))
    return code.astype(np.uint8).reshape(-1), np.where(bad, 255, e).astype(np.uint8)


def step_words(n, seed, step):
    """(for exp_avg, for exp_avg_sq): the 16-bit words of n elements, n a multiple of 256."""
    w = philox_words(np.arange(n // 8, dtype=np.uint64), seed % 2 ** 64, step, SITE).reshape(-1).astype(np.int64)
    return (w >> 8) | ((w & 255) << 8), w


def averages_f32(m, v, g, b1, b2, clip=None):
    """m', v' in float32, every product and sum rounded by itself, as the kernel takes them."""
    f = np.float32
    h = g.astype(f) if clip is None else g.astype(f) * f(clip)
    return m * f(b1) + h * f(1 - b1), v * f(b2) + (h * h) * f(1 - b2)


def adamw(p, g, m, v, t, lr, b1, b2, eps, wd, clip=1.0):
    """One step in float64: {name: (value, scale of its rounding errors)} for p, m, v; p's scale is
    (of the weight, of the step)."""
    p, g, m, v = (x.double() for x in (p, g, m, v))
    h = g * clip
    m1, v1 = b1 * m + (1 - b1) * h, b2 * v + (1 - b2) * h * h
    am = b1 * m.abs() + (1 - b1) * h.abs()
    denom = (v1 / (1 - b2 ** t)).sqrt() + eps
    rate = lr / (1 - b1 ** t)
    return {"m": (m1, am), "v": (v1, v1), "p": (p * (1 - lr * wd) - rate * m1 / denom, (p.abs(), rate * am / denom))}

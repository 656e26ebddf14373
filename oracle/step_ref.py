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

"""Float64 restatement of the training operators (oracle; test infrastructure).

Each function returns its results and, beside every result, the sum of the
absolute values of the terms it is made of: the scale that rounding errors of
the kernels' 16-bit and 32-bit steps are proportional to.
"""
from __future__ import annotations

import math

import numpy as np
import torch

Tensor = torch.Tensor


def philox_words(block: np.ndarray, seed: int, step: int, site: int) -> np.ndarray:
    """[..., 8] 16-bit words of Philox4x32 with seven rounds; counter (block, step, site), key = seed."""
    u32, m = np.uint64(32), np.uint64(0xFFFFFFFF)
    b = block.astype(np.uint64)
    c = [b & m, b >> u32, np.full_like(b, step & 0xFFFFFFFF), np.full_like(b, site & 0xFFFFFFFF)]
    k = [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF]
    for _ in range(7):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> u32) ^ c[1] ^ np.uint64(k[0]), p1 & m, (p0 >> u32) ^ c[3] ^ np.uint64(k[1]), p0 & m]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    w = np.stack(c, -1)
    return np.stack([w & np.uint64(0xFFFF), w >> np.uint64(16)], -1).reshape(*b.shape, 8)


def keep_factor(rows: int, cols: int, p: float, seed: int, step: int, site: int) -> Tensor:
    """[rows, cols] float64: 1 / (1 - p) (p in units of 2^-16) where an element stays, else 0."""
    t = round(p * 65536)
    if t == 0:
        return torch.ones(rows, cols, dtype=torch.float64)
    per = (cols + 7) // 8
    w = philox_words(np.arange(rows * per, dtype=np.uint64), seed, step, site).reshape(rows, per * 8)[:, :cols]
    return torch.from_numpy((w >= t).astype(np.float64) * (65536.0 / (65536 - t)))


def attention(q, k, v, dout, pads, scale=None, keep=None):
    """q, dout [B,S,Hq,D], k, v [B,S,Hkv,D] (any dtype, CPU); pads: B ints; keep [B,Hq,S,S] factors or None.
    Returns {name: (value, scale of its rounding errors)} for out, dq, dk, dv, and the same for the part that
    an error of delta (relative to sum |O| |dO|) adds to dq and dk under "dq_delta", "dk_delta"."""
    q, k, v, dout = (t.double() for t in (q, k, v, dout))
    B, S, Hq, D = q.shape
    Hkv = k.shape[2]
    R = Hq // Hkv
    sc = 1.0 / math.sqrt(D) if scale is None else scale
    z = {n: torch.zeros_like(t) for n, t in (("out", q), ("dq", q), ("dk", k), ("dv", v), ("dq_delta", q),
                                             ("dk_delta", k))}
    a = {n: torch.zeros_like(t) for n, t in z.items()}
    for b in range(B):
        lo = min(max(int(pads[b]), 0), S)
        if lo == S:
            continue
        n = S - lo
        causal = torch.ones(n, n, dtype=torch.bool).tril()
        for h in range(Hq):
            g = h // R
            qq, kk, vv, do = q[b, lo:, h], k[b, lo:, g], v[b, lo:, g], dout[b, lo:, h]
            s = (qq @ kk.T * sc).masked_fill(~causal, -math.inf)
            P = torch.softmax(s, -1)
            f = torch.ones(n, n, dtype=torch.float64) if keep is None else keep[b, h, lo:, lo:]
            z["out"][b, lo:, h] = (P * f) @ vv
            a["out"][b, lo:, h] = (P * f) @ vv.abs()
            z["dv"][b, lo:, g] += (P * f).T @ do
            a["dv"][b, lo:, g] += (P * f).T @ do.abs()
            dP = (do @ vv.T) * f
            dS = P * (dP - (P * dP).sum(-1, keepdim=True))
            dS[0] = 0
            z["dq"][b, lo:, h] = dS @ kk * sc
            a["dq"][b, lo:, h] = dS.abs() @ kk.abs() * sc
            z["dk"][b, lo:, g] += dS.T @ qq * sc
            a["dk"][b, lo:, g] += dS.abs().T @ qq.abs() * sc
            off = P * ((P * f) @ vv * do).abs().sum(-1, keepdim=True)
            size = P * ((do.abs() @ vv.abs().T) * f + (P * ((do.abs() @ vv.abs().T) * f)).sum(-1, keepdim=True))
            z["dq_delta"][b, lo:, h] = off @ kk.abs() * sc
            z["dk_delta"][b, lo:, g] += off.T @ qq.abs() * sc
            a["dq_delta"][b, lo:, h] = size @ kk.abs() * sc
            a["dk_delta"][b, lo:, g] += size.T @ qq.abs() * sc
    return {n: (z[n], a[n]) for n in z}


def residual_norm(x, residual, w_pre, w_post, gate, alpha, eps, keep, dh, dn):
    """x, residual, dh, dn [M,H]; gate [G,H] (G divides M) or None; keep [M,H] factors.  Returns
    {name: (value, magnitude)} for h, n, dx, dres, dpre, dpost, dgate."""
    x, w_pre, keep = x.double(), w_pre.double(), keep.double()
    M, H = x.shape
    residual, dh, dn = (torch.zeros_like(x) if t is None else t.double() for t in (residual, dh, dn))
    rows = 1 if gate is None else M // gate.shape[0]
    g = torch.full_like(x, alpha) if gate is None else alpha * gate.double().repeat_interleave(rows, 0)
    rp = torch.ones(M, 1, dtype=torch.float64)
    u = x
    if w_post is not None:
        rp = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
        u = x * rp * w_post.double()
    v = u * keep
    h = residual + g * v
    ha = residual.abs() + (g * v).abs()
    r = (h.square().mean(-1, keepdim=True) + eps).rsqrt()
    t, hh, hha = dn * w_pre, h * r, ha * r
    c, ca = (t * hh).mean(-1, keepdim=True), (t.abs() * hha).mean(-1, keepdim=True)
    d = dh + r * (t - hh * c)
    da = dh.abs() + r * (t.abs() + hha * ca)
    du, dua = d * g * keep, da * g.abs() * keep
    out = {"h": (h, ha), "n": (hh * w_pre, hha * w_pre.abs()), "dres": (d, da),
           "dpre": ((dn * hh).sum(0), (dn.abs() * hha).sum(0)), "dx": (du, dua), "dpost": None, "dgate": None}
    if gate is not None:
        out["dgate"] = tuple(z.view(-1, rows, H).sum(1) for z in (alpha * v * d, abs(alpha) * v.abs() * da))
    if w_post is not None:
        xh, s, sa = x * rp, du * w_post.double(), dua * w_post.double().abs()
        out["dpost"] = ((du * xh).sum(0), (dua * xh.abs()).sum(0))
        c, ca = (s * xh).mean(-1, keepdim=True), (sa * xh.abs()).mean(-1, keepdim=True)
        out["dx"] = (rp * (s - xh * c), rp * (sa + xh.abs() * ca))
    return out

"""Training operators of the Decision Transformer block: cases, plain forms and the framework's calls.

Three operators make one training step of a block: causal grouped-query attention with its gradient
(``attn``), the residual add with its norms, gate and dropout and their gradients (``norm``), and the
stand-alone dropout (``drop``).  Every pass is forward and backward; a mask of dropout is never an
input or an output: it is a function of (seed, step, site, element) that both directions evaluate.
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


# ------------------------------------------------------------------------------------------ cases
def _attn(name, batch, seq, heads, kv_heads, dim, dtype, p, pad_max):
    return {"name": name, "op": "attn", "batch": batch, "seq": seq, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "dtype": dtype, "p": p, "pad_max": pad_max}


def _norm(name, batch, seq, hidden, dtype, post, gate, p):
    return {"name": name, "op": "norm", "batch": batch, "seq": seq, "hidden": hidden, "dtype": dtype,
            "post": post, "gate": gate, "p": p}


def _drop(name, rows, hidden, dtype, residual, p):
    return {"name": name, "op": "drop", "rows": rows, "hidden": hidden, "dtype": dtype, "residual": residual,
            "p": p}


def listed():
    return [
        # The first timestep of one episode (return, state, action): launch latency only.
        _attn("attn one timestep", 1, 3, 8, 2, 32, "bf16", 0.1, 0),
        # A training batch of the default model: 64 left-padded contexts of 64 timesteps, dropout 0.1.
        _attn("attn default batch", 64, 192, 8, 2, 32, "bf16", 0.1, 96),
        # The same contexts at the batch the attention benchmark uses half of, fine-tuning without dropout.
        _attn("attn many contexts", 2048, 192, 8, 2, 32, "bf16", 0.0, 96),
        # The larger model: 256 timesteps, 12 / 4 heads of 64, dropout 0.1, padding up to 128 timesteps.
        _attn("attn large model", 96, 768, 12, 4, 64, "bf16", 0.1, 384),
        # A whole episode as one context, of odd length, fp16, every head with its own keys.
        _attn("attn whole episode", 1, 5003, 12, 12, 64, "fp16", 0.0, 0),
        # One timestep of one episode through the residual add and the next norm: latency only.
        _norm("norm one timestep", 1, 3, 256, "bf16", False, "none", 0.1),
        # The default model's residual add + dropout + next block's norm on a training batch.
        _norm("norm default batch", 64, 192, 256, "bf16", False, "none", 0.1),
        # The larger model with norms on both sides of the block and a learned gate of each channel.
        _norm("norm large model", 96, 768, 768, "bf16", True, "channel", 0.0),
        # fp32, an odd width, and a gate of each sample (conditioning on the episode), with dropout.
        _norm("norm odd fp32", 33, 129, 1001, "fp32", True, "sample", 0.1),
        # One context's projection output with its residual: latency only.
        _drop("drop one context", 192, 256, "bf16", True, 0.1),
        # The larger model's feed-forward activations of a training batch.
        _drop("drop large model", 73728, 2048, "bf16", False, 0.1),
        # fp32 rows of an odd width, added to their residual.
        _drop("drop odd fp32", 12289, 1001, "fp32", True, 0.25),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attn", "attn", "norm", "drop"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    p = rng.choice([0.0, 0.1, round(rng.uniform(0.01, 0.5), 3)])
    if op == "attn":
        dim = rng.choice([32, 64])
        kv_heads = rng.choice([1, 2, 3, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 3, 4] if kv_heads <= 4 else [1, 2])
        seq = _log(rng, 1, 4900)
        # The products stay under the large model's, the bytes under the many contexts'.
        most = min(3.85e8 / (heads * seq * seq), 3.0e6 / (heads * seq), 4096)
        batch = _log(rng, 1, max(1.0, most))
        pad_max = rng.choice([0, seq // 2, seq])
        return {"op": op, "batch": batch, "seq": seq, "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "dtype": dtype, "p": p, "pad_max": pad_max}
    dtype = rng.choice(["bf16", "fp16", "fp32"])
    if op == "norm":
        hidden = rng.choice([_log(rng, 32, 4096), 8 * _log(rng, 4, 512)])
        tokens = _log(rng, 1, min(70000.0, 5.0e7 / hidden))
        seq = min(tokens, rng.choice([1, 3, 189, 192, 255, 768]))
        return {"op": op, "batch": max(1, tokens // seq), "seq": seq, "hidden": hidden, "dtype": dtype,
                "post": rng.random() < 0.5, "gate": rng.choice(["none", "channel", "sample", "token"]), "p": p}
    hidden = rng.choice([_log(rng, 32, 4096), 8 * _log(rng, 4, 512)])
    rows = _log(rng, 1, min(70000.0, 1.2e8 / hidden))
    return {"op": op, "rows": rows, "hidden": hidden, "dtype": dtype, "residual": rng.random() < 0.5,
            "p": rng.choice([0.1, round(rng.uniform(0.01, 0.9), 3)])}


# ----------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _TYPES[case["dtype"]]

    def randn(*shape, scale=1.0, shift=0.0):
        return torch.randn(*shape, generator=g, device="cuda").mul_(scale).add_(shift).to(dt)

    s = {"case": case, "p": case["p"], "site": 1 + seed % 7}
    # The generator's state as a training loop keeps it: seed and step on the device.
    s["rng"] = torch.randint(0, 2 ** 31 - 1, (2,), generator=g, device="cuda")
    if case["op"] == "attn":
        B, S, Hq, Hkv, D = (case[k] for k in ("batch", "seq", "heads", "kv_heads", "dim"))
        # q | k | v as the projection writes them: views of one tensor.
        qkv = randn(B, S, Hq + 2 * Hkv, D)
        s["q"], s["k"], s["v"] = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hkv], qkv[:, :, Hq + Hkv:]
        s["dout"] = randn(B, S, Hq, D)
        s["pad"] = None
        if case["pad_max"]:
            s["pad"] = torch.randint(0, case["pad_max"] + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
        return s
    if case["op"] == "norm":
        B, S, H = case["batch"], case["seq"], case["hidden"]
        s["x"], s["residual"] = randn(B, S, H), randn(B, S, H, scale=2.0)
        s["w_pre"] = randn(H, scale=0.1, shift=1.0)
        s["w_post"] = randn(H, scale=0.1, shift=1.0) if case["post"] else None
        shape = {"none": None, "channel": (H,), "sample": (B, 1, H), "token": (B, S, H)}[case["gate"]]
        s["gate"] = None if shape is None else randn(*shape, scale=0.3, shift=0.5)
        s["alpha"] = 0.7 if case["gate"] != "none" else 1.0
        s["dh"], s["dn"] = randn(B, S, H), randn(B, S, H)
        return s
    s["x"] = randn(case["rows"], case["hidden"])
    s["residual"] = randn(case["rows"], case["hidden"]) if case["residual"] else None
    s["dy"] = randn(case["rows"], case["hidden"])
    return s


EPS = 1e-5


# ------------------------------------------------------------------------------------ plain forms
def _philox_words(block, rng, site):
    """The eight 16-bit words of each counter block: Philox4x32 with seven rounds (Salmon, Moraes,
    Dror, Shaw, SC 2011), counter (block, step, site), key = seed; int64 [..., 8]."""
    low = 0xFFFFFFFF
    seed, step = rng[0], rng[1]
    c0, c1 = block & low, (block >> 32) & low
    c2 = (step & low).expand_as(c0)
    c3 = torch.full_like(c0, site)
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(7):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    w = torch.stack((c0, c1, c2, c3), -1)
    return torch.stack((w & 0xFFFF, w >> 16), -1).flatten(-2)


def _keep(rows, cols, p, rng, site):
    """[rows, cols] float32: 1 / (1 - p) where an element stays, 0 where it is dropped; each row starts
    a new block of eight words."""
    threshold = int(round(p * 65536))
    per_row = (cols + 7) // 8
    block = torch.arange(rows * per_row, device=rng.device)
    w = _philox_words(block, rng, site).view(rows, per_row * 8)[:, :cols]
    return (w >= threshold).float() * (65536.0 / (65536 - threshold))


def _attn_plain(s):
    q, k, v, dout, pad = s["q"], s["k"], s["v"], s["dout"], s["pad"]
    B, S, Hq, D = q.shape
    Hkv = k.shape[2]
    R = Hq // Hkv
    scale = 1.0 / math.sqrt(D)
    qf = q.float().permute(0, 2, 1, 3).reshape(B, Hkv, R, S, D)
    dof = dout.float().permute(0, 2, 1, 3).reshape(B, Hkv, R, S, D)
    kf = k.float().permute(0, 2, 1, 3).unsqueeze(2)
    vf = v.float().permute(0, 2, 1, 3).unsqueeze(2)
    at = torch.arange(S, device=q.device)
    seen = (at[None, :] <= at[:, None])[None]
    if pad is not None:
        seen = seen & (at[None, None, :] >= pad[:, None, None])
    seen = seen[:, None, None]
    sc = torch.matmul(qf, kf.transpose(-1, -2)).mul_(scale).masked_fill_(~seen, -math.inf)
    top = sc.amax(-1, keepdim=True)
    e = torch.exp(sc.sub_(top.masked_fill(top == -math.inf, 0.0)))
    total = e.sum(-1, keepdim=True)
    prob = e / total.masked_fill(total == 0, 1.0)
    if s["p"] > 0:
        keep = _keep(B * Hq * S, S, s["p"], s["rng"], s["site"]).view(B, Hkv, R, S, S)
        dropped = prob * keep
    else:
        dropped = prob
    out = torch.matmul(dropped, vf)
    dv = torch.matmul(dropped.transpose(-1, -2), dof).sum(2)
    dp = torch.matmul(dof, vf.transpose(-1, -2))
    if s["p"] > 0:
        dp = dp * keep
    ds = prob * (dp - (prob * dp).sum(-1, keepdim=True)) * scale
    dq = torch.matmul(ds, kf)
    dk = torch.matmul(ds.transpose(-1, -2), qf).sum(2)
    out, dq = (t.reshape(B, Hq, S, D).permute(0, 2, 1, 3) for t in (out, dq))
    return {"out": out.to(q.dtype), "dq": dq.to(q.dtype), "dk": dk.permute(0, 2, 1, 3).to(q.dtype),
            "dv": dv.permute(0, 2, 1, 3).to(q.dtype)}


def _norm_plain(s):
    x, res, dh, dn = (s[k].float() for k in ("x", "residual", "dh", "dn"))
    dt, alpha = s["x"].dtype, s["alpha"]
    B, S, H = x.shape
    wpre = s["w_pre"].float()
    y, xhat = x, None
    if s["w_post"] is not None:
        wpost = s["w_post"].float()
        rpost = torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + EPS)
        xhat = x * rpost
        y = xhat * wpost
    keep = _keep(B * S, H, s["p"], s["rng"], s["site"]).view(B, S, H) if s["p"] > 0 else None
    y = y * keep if keep is not None else y
    gate = alpha if s["gate"] is None else alpha * s["gate"].float()
    h = res + gate * y
    rpre = torch.rsqrt(h.pow(2).mean(-1, keepdim=True) + EPS)
    hhat = h * rpre
    out = {"h": h.to(dt), "n": (hhat * wpre).to(dt)}
    out["dw_pre"] = (dn * hhat).sum((0, 1)).to(dt)
    t = dn * wpre
    dt_h = dh + rpre * (t - hhat * (t * hhat).mean(-1, keepdim=True))
    out["dresidual"] = dt_h.to(dt)
    if s["gate"] is not None:
        dg = alpha * y * dt_h
        over = {"channel": (0, 1), "sample": (1,), "token": ()}[s["case"]["gate"]]
        out["dgate"] = (dg.sum(over, keepdim=len(over) == 1) if over else dg).to(dt)
    dy = gate * dt_h
    dy = dy * keep if keep is not None else dy
    if s["w_post"] is not None:
        out["dw_post"] = (dy * xhat).sum((0, 1)).to(dt)
        t = dy * wpost
        dy = rpost * (t - xhat * (t * xhat).mean(-1, keepdim=True))
    out["dx"] = dy.to(dt)
    return out


def _drop_plain(s):
    x, dt = s["x"], s["x"].dtype
    keep = _keep(x.shape[0], x.shape[1], s["p"], s["rng"], s["site"])
    y = x.float() * keep
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return {"y": y.to(dt), "dx": (s["dy"].float() * keep).to(dt)}


# -------------------------------------------------------------------------------------- own calls
def _attn_own(s):
    from rl_for_mario_b200 import kernels

    out, lse = kernels.attn_train_forward(s["q"], s["k"], s["v"], s["pad"], p=s["p"], rng=s["rng"], site=s["site"])
    dq, dk, dv = kernels.attn_train_backward(s["dout"], s["q"], s["k"], s["v"], out, lse, s["pad"], p=s["p"],
                                             rng=s["rng"], site=s["site"])
    return {"out": out, "dq": dq, "dk": dk, "dv": dv}


def _norm_own(s):
    from rl_for_mario_b200 import kernels

    how = dict(post_weight=s["w_post"], gate=s["gate"], alpha=s["alpha"], p=s["p"], rng=s["rng"], site=s["site"])
    h, n, stats = kernels.residual_norm_forward(s["x"], s["residual"], s["w_pre"], EPS, **how)
    dx, dres, dpre, dpost, dgate = kernels.residual_norm_backward(s["dh"], s["dn"], s["x"], s["residual"],
                                                                  s["w_pre"], stats, **how)
    out = {"h": h, "n": n, "dw_pre": dpre, "dresidual": dres, "dx": dx}
    if dgate is not None:
        out["dgate"] = dgate
    if dpost is not None:
        out["dw_post"] = dpost
    return out


def _drop_own(s):
    from rl_for_mario_b200 import kernels

    y = kernels.dropout_forward(s["x"], s["p"], s["rng"], site=s["site"], residual=s["residual"])
    return {"y": y, "dx": kernels.dropout_backward(s["dy"], s["p"], s["rng"], site=s["site"])}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"attn": _attn_own, "norm": _norm_own, "drop": _drop_own}[op](state)
    return {"attn": _attn_plain, "norm": _norm_plain, "drop": _drop_plain}[op](state)


# ------------------------------------------------------------------------------------------- work
def work(case):
    e = _SIZE[case["dtype"]]
    if case["op"] == "attn":
        B, S, Hq, Hkv, D = (case[k] for k in ("batch", "seq", "heads", "kv_heads", "dim"))
        # Rows behind the padding attend to nothing: a valid row q to q - pad + 1 keys, mean over the pads.
        pads = case["pad_max"]
        step = max(1, pads // 64)
        lens = [S - a for a in range(0, pads + 1, step)]
        pairs = B * Hq * sum(n * (n + 1) / 2 for n in lens) / len(lens)
        # read q, k, v, dout; write out, dq, dk, dv; two products forward, five backward.
        return {"bytes": e * B * S * D * (4 * Hq + 4 * Hkv), "flops": 7 * 2 * D * pairs}
    if case["op"] == "norm":
        B, S, H = case["batch"], case["seq"], case["hidden"]
        per = 8  # x, residual, dh, dn in; h, n, dx, dresidual out
        if case["gate"] == "token":
            per += 2
        small = {"none": 0, "channel": 2 * H, "sample": 2 * B * H, "token": 0}[case["gate"]] + H * (4 if case["post"] else 2)
        return {"bytes": e * (per * B * S * H + small), "flops": 30 * B * S * H}
    n = case["rows"] * case["hidden"]
    return {"bytes": e * n * (5 if case["residual"] else 4), "flops": 4 * n}


# ------------------------------------------------------------------------------------------ exact
def _stays(index, seed, step, site, p):
    """Whether the elements with these (block * 8 + word) indices stay, by the definition of the
    generator, products taken in 16-bit halves."""
    m = 2 ** 32

    def mul(c, x):
        lo, hi = x % 65536, x // 65536
        a, b = lo * c, hi * c                       # both below 2^48
        t = a + (b % 65536) * 65536
        return (b // 65536 + t // m) % m, t % m     # high and low words

    block, word = index // 8, index % 8
    x = [block % m, block // m, torch.full_like(block, step % m), torch.full_like(block, site)]
    key = [seed % m, seed // m]
    for r in range(7):
        h0, l0 = mul(0xD2511F53, x[0])
        h1, l1 = mul(0xCD9E8D57, x[2])
        x = [h1 ^ x[1] ^ ((key[0] + r * 0x9E3779B9) % m), l1, h0 ^ x[3] ^ ((key[1] + r * 0xBB67AE85) % m), l0]
    which = word // 2
    v = torch.where(which == 0, x[0], torch.where(which == 1, x[1], torch.where(which == 2, x[2], x[3])))
    v = torch.where(word % 2 == 0, v % 65536, v // 65536)
    return v >= int(round(p * 65536))


def _factor(s, first, rows, cols):
    """float64 [rows, cols] dropout factors of rows first .. first + rows."""
    seed, step = (int(t) for t in s["rng"].tolist())
    r = torch.arange(first, first + rows, device="cuda")[:, None]
    c = torch.arange(cols, device="cuda")[None, :]
    index = (r * ((cols + 7) // 8) + c // 8) * 8 + c % 8
    t = int(round(s["p"] * 65536))
    return _stays(index, seed, step, s["site"], s["p"]).double() * 65536 / (65536 - t)


def _attn_exact(s):
    q, k, v, dout = (s[n].double() for n in ("q", "k", "v", "dout"))
    B, S, Hq, D = q.shape
    Hkv = k.shape[2]
    R = Hq // Hkv
    out, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    pads = [0] * B if s["pad"] is None else s["pad"].tolist()
    for b in range(B):
        a = pads[b]
        n = S - a
        if n < 1:
            continue
        for h in range(Hq):
            g = h // R
            logits = q[b, a:, h] @ k[b, a:, g].T / D ** 0.5
            logits = logits + torch.full((n, n), -math.inf, dtype=torch.float64, device="cuda").triu(1)
            prob = torch.softmax(logits, -1)
            f = torch.ones((), dtype=torch.float64, device="cuda")
            if s["p"] > 0:
                f = _factor(s, (b * Hq + h) * S + a, n, S)[:, a:]
            do = dout[b, a:, h]
            out[b, a:, h] = (prob * f) @ v[b, a:, g]
            dv[b, a:, g] += (prob * f).T @ do
            dprob = (do @ v[b, a:, g].T) * f
            dlogits = prob * (dprob - (prob * dprob).sum(-1, keepdim=True))
            dq[b, a:, h] = dlogits @ k[b, a:, g] / D ** 0.5
            dk[b, a:, g] += dlogits.T @ q[b, a:, h] / D ** 0.5
    return {"out": out, "dq": dq, "dk": dk, "dv": dv}


def _norm_exact(s):
    shape = s["x"].shape
    x, res, dh, dn = (s[k].double().reshape(-1, shape[-1]) for k in ("x", "residual", "dh", "dn"))
    M, H = x.shape
    wpre = s["w_pre"].double()
    gate = torch.full_like(x, s["alpha"])
    if s["gate"] is not None:
        gate = s["alpha"] * s["gate"].double().expand(shape).reshape(M, H)
    f = _factor(s, 0, M, H) if s["p"] > 0 else torch.ones_like(x)
    xn, a = x, None
    if s["w_post"] is not None:
        a = (x.square().sum(-1, keepdim=True) / H + EPS).sqrt()
        xn = s["w_post"].double() * x / a
    h = res + gate * f * xn
    c = (h.square().sum(-1, keepdim=True) / H + EPS).sqrt()
    # n_i = w_i h_i / c, dc / dh_i = h_i / (H c)
    total = dh + dn * wpre / c - h * (dn * wpre * h).sum(-1, keepdim=True) / (H * c ** 3)
    out = {"h": h.view(shape), "n": (wpre * h / c).view(shape), "dw_pre": (dn * h / c).sum(0),
           "dresidual": total.view(shape)}
    if s["gate"] is not None:
        dg = (total * s["alpha"] * f * xn).view(shape)
        out["dgate"] = {"channel": lambda: dg.sum((0, 1)), "sample": lambda: dg.sum(1, keepdim=True),
                        "token": lambda: dg}[s["case"]["gate"]]()
    dxn = total * gate * f
    if s["w_post"] is not None:
        wpost = s["w_post"].double()
        out["dw_post"] = (dxn * x / a).sum(0)
        dxn = dxn * wpost / a - x * (dxn * wpost * x).sum(-1, keepdim=True) / (H * a ** 3)
    out["dx"] = dxn.view(shape)
    return out


def _drop_exact(s):
    x = s["x"]
    f = _factor(s, 0, x.shape[0], x.shape[1])
    y = x.double() * f
    if s["residual"] is not None:
        y += s["residual"].double()
    return {"y": y, "dx": s["dy"].double() * f}


def exact(case, seed):
    if case["op"] == "attn" and case["batch"] * case["heads"] > (8000 if case["p"] > 0 else 16384):
        return None  # one product at a time over every head: too long
    s = prepare(case, seed)
    return {"attn": _attn_exact, "norm": _norm_exact, "drop": _drop_exact}[case["op"]](s)

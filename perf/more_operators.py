"""Operators of a training step around its products: cases, plain forms and the framework's calls.

``heads``: the norm of every query and key head with the position rotation in the same pass, with its
gradient (training) or without (a rollout's new tokens).  ``norm``: the norm of a whole model's gradient.
``adamw``: an AdamW step over all of a model's tensors, clipped by that norm, with its averages in 32 or in
8 bits.  The 8-bit averages are blocks of 256 elements with a power of two as their scale, rounded up or down
at random by words that are a function of (seed, step, element).
"""
import math
import random

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}

EPS = 1e-5                              # of the norms
LR, B1, B2, ADAM_EPS = 3e-4, 0.9, 0.999, 1e-8
DECAY = 0.1                             # of matrices; vectors have none
BLOCK = 256                             # elements that share a scale; every tensor starts a new block
SITE = 2 ** 32 - 1                      # the generator's site of the averages' rounding
# The averages in 8 bits: exponent bias, exponent of a block's largest value, whether there is a sign.  The first are
# numbers of four exponent bits, the second of five, both of three behind the leading one.
FIRST, SECOND = (7, 7, True), (15, 14, False)


# ------------------------------------------------------------------------------------------ cases
def _heads(name, batch, seq, heads, kv_heads, dim, dtype, train, starts):
    return {"name": name, "op": "heads", "batch": batch, "seq": seq, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "dtype": dtype, "train": train, "starts": starts}


def _model(name, op, hidden, layers, kv_width, inter, positions, dtype, bits=32, master=False, clip=False):
    return {"name": name, "op": op, "kind": "model", "hidden": hidden, "layers": layers, "kv_width": kv_width,
            "inter": inter, "positions": positions, "dtype": dtype, "bits": bits, "master": master, "clip": clip}


def _some(name, op, tensors, least, most, mix, dtype, bits=32, master=False, clip=False):
    return {"name": name, "op": op, "kind": "some", "tensors": tensors, "least": least, "most": most, "mix": mix,
            "dtype": dtype, "bits": bits, "master": master, "clip": clip}


def listed():
    return [
        # The first timestep of one episode (return, state, action) in training: launch latency only.
        _heads("heads one timestep", 1, 3, 8, 2, 32, "bf16", True, False),
        # A training batch of the default model.
        _heads("heads default batch", 64, 192, 8, 2, 32, "bf16", True, False),
        # The larger model: 256 timesteps, 12 / 4 heads of 64.
        _heads("heads large model", 96, 768, 12, 4, 64, "bf16", True, False),
        # fp32, heads of an uneven width, every query head with its own keys.
        _heads("heads odd fp32", 33, 129, 5, 5, 42, "fp32", True, False),
        # A rollout step of 16,384 environments: three new tokens each, every one at its own position.
        _heads("heads rollout step", 16384, 3, 8, 2, 32, "bf16", False, True),
        # The gradient of the default model under autocast.
        _model("norm default model", "norm", 256, 4, 64, 704, 4096, "fp32"),
        # The larger model's in 16 bits.
        _model("norm large model", "norm", 768, 12, 256, 2048, 4096, "bf16"),
        # Fine-tuning the two heads of a frozen model alone: four tensors, latency only.
        _some("adamw heads only", "adamw", 4, 1, 2048, 1, "fp32"),
        # The default model in fp32 (trained under autocast), clipped.
        _model("adamw default model", "adamw", 256, 4, 64, 704, 4096, "fp32", clip=True),
        # The larger model in 16 bits with fp32 weights beside it, clipped.
        _model("adamw large master", "adamw", 768, 12, 256, 2048, 4096, "bf16", master=True, clip=True),
        # The larger model in 16 bits, its averages in 8, clipped.
        _model("adamw large 8 bits", "adamw", 768, 12, 256, 2048, 4096, "bf16", bits=8, clip=True),
        # Many tensors of odd sizes in fp32 with averages in 8 bits.
        _some("adamw odd 8 bits", "adamw", 61, 1, 300001, 7, "fp32", bits=8),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["heads", "heads", "norm", "adamw", "adamw"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "heads":
        dim = rng.choice([32, 64, 32, 64, 16, 128, 256, 2 * _log(rng, 1, 128)])
        kv_heads = rng.choice([1, 2, 3, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 3, 4] if kv_heads <= 4 else [1, 2])
        train = rng.random() < 0.65
        tokens = _log(rng, 1, max(1.0, min(70000.0, 7.0e7 / ((heads + kv_heads) * dim))))
        seq = min(tokens, rng.choice([1, 2, 3, 189, 192, 255, 768, 5003]) if train else rng.choice([1, 2, 3, 6]))
        return {"op": op, "batch": max(1, tokens // seq), "seq": seq, "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "dtype": dtype, "train": train, "starts": rng.random() < (0.25 if train else 0.75)}
    bits = 32 if op == "norm" else rng.choice([32, 8])
    how = {"dtype": dtype, "bits": bits, "master": op == "adamw" and dtype != "fp32" and rng.random() < 0.5,
           "clip": op == "adamw" and rng.random() < 0.5}
    if rng.random() < 0.5:
        heads, dim, layers = rng.choice([2, 3, 4, 6, 8, 12]), rng.choice([32, 64]), _log(rng, 1, 10)
        return {"op": op, "kind": "model", "hidden": heads * dim, "layers": layers, "kv_width": dim * rng.choice([1, 2]),
                "inter": 64 * _log(rng, 1, 32), "positions": _log(rng, 16, 4096), **how}
    tensors = _log(rng, 1, 160)
    most = _log(rng, 1, min(4.0e6, 6.0e7 / tensors))
    return {"op": op, "kind": "some", "tensors": tensors, "least": _log(rng, 1, most), "most": most,
            "mix": rng.randrange(1000), **how}


def _shapes(case):
    """The tensors' shapes, matrices first (they decay), then vectors."""
    if case["kind"] == "model":
        h, kv, inter = case["hidden"], case["kv_width"], case["inter"]
        first = [(32, 4, 8, 8), (64, 32, 4, 4), (64, 64, 3, 3), (h, 3136), (h, 1), (7, h), (case["positions"], h)]
        block = [(h, h), (kv, h), (kv, h), (h, h), (inter, h), (inter, h), (h, inter)]
        matrices = first + block * case["layers"] + [(7, h), (1, h)]
        return matrices, [(32,), (64,), (64,), (h,), (h,), (h,)] + [(h,), (h,)] * case["layers"] + [(h,), (1,)]
    rng = random.Random(case["mix"])
    lo, hi = sorted((case["least"], case["most"]))
    sizes = [_log(rng, lo, hi) for _ in range(case["tensors"])]
    return [(n,) for n in sizes[: len(sizes) // 2]], [(n,) for n in sizes[len(sizes) // 2:]]


def _up(n):
    return (n + BLOCK - 1) // BLOCK * BLOCK


# ----------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _TYPES[case["dtype"]]

    def randn(*shape, scale=1.0, shift=0.0):
        return torch.randn(*shape, generator=g, device="cuda").mul_(scale).add_(shift)

    s = {"case": case}
    if case["op"] == "heads":
        B, S, Hq, Hkv, D = (case[k] for k in ("batch", "seq", "heads", "kv_heads", "dim"))
        # q | k | v as the projection writes them: q and k are views of one tensor.
        qkv = (randn(B, S, Hq + 2 * Hkv, D) * torch.exp(randn(B, S, 1, 1, scale=0.5))).to(dt)
        s["q"], s["k"] = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hkv]
        s["wq"], s["wk"] = randn(D, scale=0.1, shift=1.0).to(dt), randn(D, scale=0.1, shift=1.0).to(dt)
        rows = S + (4096 if case["starts"] else 0)
        angle = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] / 1e4 ** (
            torch.arange(0, D, 2, device="cuda", dtype=torch.float64) / D)
        s["cos"], s["sin"] = (f(angle).float().repeat(1, 2) for f in (torch.cos, torch.sin))
        s["start"] = None
        if case["starts"]:
            s["start"] = torch.randint(0, 4097, (B,), generator=g, device="cuda", dtype=torch.int32)
        if case["train"]:
            s["dq"], s["dk"] = randn(B, S, Hq, D).to(dt), randn(B, S, Hkv, D).to(dt)
        return s
    matrices, vectors = _shapes(case)
    shapes = matrices + vectors
    at = [0]
    for shape in shapes:
        at.append(at[-1] + _up(math.prod(shape)))
    split = at[len(matrices)]  # where the vectors begin
    live = torch.zeros(at[-1], dtype=torch.bool, device="cuda")
    for a, shape in zip(at, shapes):
        live[a:a + math.prod(shape)] = True
    # A block's gradients have a size of their own; most steps have to be clipped to 1.
    size = torch.exp(randn(at[-1] // BLOCK, 1)).expand(-1, BLOCK).reshape(-1).mul_(live)

    def views(flat):
        return [flat[a:a + math.prod(shape)].view(shape) for a, shape in zip(at, shapes)]

    s["grad"] = randn(at[-1], scale=2e-3).mul_(size).to(dt)
    s["grads"] = views(s["grad"])
    if case["op"] == "norm":
        return s
    s["param"] = randn(at[-1], scale=0.02).mul_(live).to(dt)
    s["params"], s["split"], s["matrices"] = views(s["param"]), split, len(matrices)
    s["master"] = None
    if case["master"]:  # fp32 weights whose rounding the 16-bit ones are
        s["master"] = s["param"].float() * (1 + 2.0 ** -13 * randn(at[-1]).clamp_(-1, 1))
        s["param"].copy_(s["master"])
    s["seed"] = seed * 7919 + 12345
    s["step"] = torch.full((), 50 + seed % 5000, dtype=torch.int64, device="cuda")
    m, v = randn(at[-1], scale=5e-4).mul_(size), (randn(at[-1]).square_().add_(0.3).mul_(2e-6)).mul_(size).mul_(size)
    if case["bits"] == 8:
        half = torch.full((at[-1] // BLOCK, BLOCK), 32768, dtype=torch.int32, device="cuda")
        s["m"], s["m_scale"], s["v"], s["v_scale"] = *_encode(m, half, *FIRST), *_encode(v, half, *SECOND)
    else:
        s["m"], s["v"] = m, v
    return s


# ------------------------------------------------------------------------------------ plain forms
def _turn(y, cos, sin):
    half = y.shape[-1] // 2
    return y * cos + torch.cat((-y[..., half:], y[..., :half]), -1) * sin


def _head_plain(x, w, cos, sin, dout):
    """(out, dx, dw) of one kind of head; the last two None without dout."""
    dt, half = x.dtype, x.shape[-1] // 2
    x, w32 = x.float(), w.float()
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    xhat = x * r
    out = _turn(xhat * w32, cos, sin).to(dt)
    if dout is None:
        return out, None, None
    dout = dout.float()
    t = dout * sin
    dy = dout * cos + torch.cat((t[..., half:], -t[..., :half]), -1)
    dw = (dy * xhat).sum((0, 1, 2), dtype=torch.float64).to(w.dtype)
    t = dy * w32
    return out, (r * (t - xhat * (t * xhat).mean(-1, keepdim=True))).to(dt), dw


def _heads_plain(s):
    B, S = s["q"].shape[:2]
    rows = torch.arange(S, device="cuda")[None]
    if s["start"] is not None:
        rows = rows + s["start"][:, None]
    cos, sin = s["cos"][rows][:, :, None], s["sin"][rows][:, :, None]
    train = s["case"]["train"]
    q, dq, dwq = _head_plain(s["q"], s["wq"], cos, sin, s["dq"] if train else None)
    k, dk, dwk = _head_plain(s["k"], s["wk"], cos, sin, s["dk"] if train else None)
    return {"q": q, "k": k, "dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk} if train else {"q": q, "k": k}


def _norm_plain(flat):
    return flat.double().square().sum().sqrt().float()


def _words(n, seed, step):
    """int64 [n]: the 16-bit word of each element: Philox4x32 with seven rounds (Salmon, Moraes, Dror, Shaw,
    SC 2011), counter (element / 8, step, site), key = seed, eight words a call."""
    low = 0xFFFFFFFF
    block = torch.arange(n // 8, device="cuda")
    c0, c1 = block & low, block >> 32
    c2 = (step & low).expand_as(c0)
    c3 = torch.full_like(c0, SITE)
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(7):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    w = torch.stack((c0, c1, c2, c3), -1)
    return torch.stack((w & 0xFFFF, w >> 16), -1).flatten()


def _two_to(k):
    return ((k + 127) << 23).to(torch.int32).view(torch.float32)


def _encode(x, words, bias, top, signed):
    """(codes, scales), uint8 [blocks, 256] and [blocks]: x rounded to three bits behind the leading one, down or
    up by its word.  A block's scale is the (biased) exponent e of its largest value, 32 at least; its codes hold
    |x| 2^(127 + top - e) with exponents from 1 - bias, subnormal numbers below; the sign is bit 7 of a signed code.
    An unsigned code is 0 for a zero alone."""
    x = x.view(-1, BLOCK)
    e = (x.abs().view(torch.int32) >> 23).amax(1, keepdim=True).clamp_(min=32)
    y = x.abs() * _two_to(127 + top - e)
    small = ((y * 2.0 ** (bias + 18)).to(torch.int32) + words) >> 16
    large = ((y.view(torch.int32) + (words << 4)) >> 20) - ((127 - bias) << 3)
    code = torch.where(y < 2.0 ** (1 - bias), small, large)
    if signed:
        code = code | ((x.view(torch.int32) >> 31) & 1) << 7
    else:
        code = torch.maximum(code, (x > 0).int())
    return code.to(torch.uint8), e[:, 0].to(torch.uint8)


def _decode(code, scale, bias, top, signed):
    if signed:
        y = code.view(torch.float8_e4m3fn).float()
    else:
        y = (code.short() << 7).view(torch.float16).float()
    return y * _two_to(scale.int()[:, None] - (127 + top))


def _part_plain(p, m, v, g, decay, c1, c2):
    """AdamW on part of the flat tensors: (p, m, v) in 32 bits."""
    m = m * B1 + g * (1 - B1)
    v = v * B2 + (g * g) * (1 - B2)
    return p * (1 - LR * decay) - (LR / c1).float() * (m / (v.sqrt() / c2.sqrt().float() + ADAM_EPS)), m, v


def _adamw_plain(s):
    case, cut = s["case"], s["split"]
    g, norm = s["grad"].float(), None
    if case["clip"]:
        norm = _norm_plain(s["grad"])
        g = g * (1.0 / (norm + 1e-6)).clamp(max=1.0)
    s["step"] += 1
    t = s["step"].double()
    c1, c2 = 1 - B1 ** t, 1 - B2 ** t
    m, v = s["m"], s["v"]
    if case["bits"] == 8:
        m, v = _decode(m, s["m_scale"], *FIRST).view(-1), _decode(v, s["v_scale"], *SECOND).view(-1)
    p = s["param"].float() if s["master"] is None else s["master"]
    both = [_part_plain(p[a], m[a], v[a], g[a], decay, c1, c2) for a, decay in ((slice(0, cut), DECAY),
                                                                             (slice(cut, None), 0.0))]
    p, m, v = (torch.cat(x) for x in zip(*both))
    s["param"].copy_(p)
    if s["master"] is not None:
        s["master"].copy_(p)
    if case["bits"] == 8:
        w = _words(m.numel(), s["seed"], s["step"]).to(torch.int32).view(-1, BLOCK)
        # One word serves both: the first average takes its bytes turned over.
        s["m"], s["m_scale"] = _encode(m, (w >> 8) | (w & 255) << 8, *FIRST)
        s["v"], s["v_scale"] = _encode(v, w, *SECOND)
        m, v = _decode(s["m"], s["m_scale"], *FIRST), _decode(s["v"], s["v_scale"], *SECOND)
        m, v = m.view(-1).bfloat16(), v.view(-1).bfloat16()  # (bf16 holds each of these values)
    else:
        s["m"].copy_(m)
        s["v"].copy_(v)
        m, v = s["m"], s["v"]
    return _answer(s, m, v, norm, s["step"].clone())


def _answer(s, m, v, norm, step):
    out = {"param": s["param"], "m": m, "v": v, "step": step}
    if s["master"] is not None:
        out["master"] = s["master"]
    if norm is not None:
        out["norm"] = norm
    return out


# -------------------------------------------------------------------------------------- own calls
def _heads_own(s):
    from rl_for_mario_b200 import kernels

    how = (s["wq"], s["wk"], EPS, s["cos"], s["sin"], s["start"])
    q, k = kernels.head_norm_rope_forward(s["q"], s["k"], *how)
    if not s["case"]["train"]:
        return {"q": q, "k": k}
    dq, dk, dwq, dwk = kernels.head_norm_rope_backward(s["dq"], s["dk"], s["q"], s["k"], *how)
    return {"q": q, "k": k, "dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk}


def _norm_own(s):
    from rl_for_mario_b200 import optim

    return optim.grad_norm(s["grads"])


def _optimizer(s):
    """The optimizer that a training program makes once, resumed from the averages in hand."""
    from rl_for_mario_b200 import optim

    case, cut = s["case"], s["matrices"]
    params = [torch.nn.Parameter(p) for p in s["params"]]
    for p, g in zip(params, s["grads"]):
        p.grad = g
    groups = [{"params": params[:cut], "weight_decay": DECAY}, {"params": params[cut:], "weight_decay": 0.0}]
    opt = optim.AdamW([x for x in groups if x["params"]], lr=LR, betas=(B1, B2), eps=ADAM_EPS, state_bits=case["bits"],
                      master=case["master"], max_norm=1.0 if case["clip"] else None, seed=s["seed"])
    saved = opt.state_dict()
    saved["state"].update(step=s["step"], exp_avg=s["m"], exp_avg_sq=s["v"])
    if case["bits"] == 8:
        saved["state"].update(exp_avg_scale=s["m_scale"], exp_avg_sq_scale=s["v_scale"])
    if s["master"] is not None:
        saved["state"].update(master=s["master"])
    opt.load_state_dict(saved)
    return opt


def _adamw_own(s):
    if "optimizer" not in s:
        s["optimizer"] = _optimizer(s)
    opt = s["optimizer"]
    opt.step()
    m, v = opt.moments()
    if s["master"] is not None:
        s["master"] = opt.master
    return _answer(s, m, v, opt.norm, opt.steps())


def run(state):
    op = state["case"]["op"]
    if own:
        return {"heads": _heads_own, "norm": _norm_own, "adamw": _adamw_own}[op](state)
    if op == "norm":
        return _norm_plain(torch.cat([g.flatten() for g in state["grads"]]))
    return {"heads": _heads_plain, "adamw": _adamw_plain}[op](state)


# ------------------------------------------------------------------------------------------- work
def work(case):
    e = _SIZE[case["dtype"]]
    if case["op"] == "heads":
        n = case["batch"] * case["seq"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        # Forward reads and writes each element, backward reads it and its gradient and writes one.
        return {"bytes": e * n * (5 if case["train"] else 2), "flops": n * (36 if case["train"] else 12)}
    n = sum(math.prod(shape) for part in _shapes(case) for shape in part)
    if case["op"] == "norm":
        return {"bytes": e * n, "flops": 2 * n}
    per = e + (e + 8 if case["master"] else 2 * e)              # gradient; weights
    per += 16 if case["bits"] == 32 else 4 + 4 / BLOCK + 4       # averages; in 8 bits handed out as numbers too
    per += e if case["clip"] else 0                             # the norm comes before the first weight
    return {"bytes": per * n, "flops": 20 * n}


# ------------------------------------------------------------------------------------------ exact
def _heads_exact(s):
    outs = {}
    rows = torch.arange(s["q"].shape[1], device="cuda").expand(s["q"].shape[:2])
    if s["start"] is not None:
        rows = rows + s["start"].long()[:, None]
    cos, sin = s["cos"].double()[rows].unsqueeze(2), s["sin"].double()[rows].unsqueeze(2)
    for n in ("q", "k"):
        x, w = s[n].double().requires_grad_(), s["w" + n].double().requires_grad_()
        with torch.enable_grad():
            y = w * x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS) ** 0.5
            a, b = y.chunk(2, -1)
            (ca, cb), (sa, sb) = cos.chunk(2, -1), sin.chunk(2, -1)
            z = torch.cat((a * ca - b * sa, b * cb + a * sb), -1)
        outs[n] = z.detach()
        if s["case"]["train"]:
            outs["d" + n], outs["dw" + n] = torch.autograd.grad(z, (x, w), s["d" + n].double())
    return outs


def _random16(n, seed, step):
    """float64 [n]: the generator's words by its definition, products taken in 16-bit halves."""
    m = 2 ** 32

    def mul(c, x):
        a, b = (x % 65536) * c, (x // 65536) * c
        t = a + (b % 65536) * 65536
        return (b // 65536 + t // m) % m, t % m

    block = torch.arange(n // 8, device="cuda")
    x = [block % m, block // m, torch.full_like(block, step % m), torch.full_like(block, SITE)]
    for r in range(7):
        h0, l0 = mul(0xD2511F53, x[0])
        h1, l1 = mul(0xCD9E8D57, x[2])
        x = [h1 ^ x[1] ^ ((seed + r * 0x9E3779B9) % m), l1, h0 ^ x[3] ^ ((seed // m + r * 0xBB67AE85) % m), l0]
    return torch.stack([f for c in x for f in (c % 65536, c // 65536)], -1).reshape(-1)


def _rounded(x, u, lowest, top):
    """x in blocks, rounded at random to three bits behind the leading one: up where the part cut off and u / 2^16
    come to a step or more.  The steps end at 2^lowest under a block's top binade, which is 2^top."""
    x = x.view(-1, BLOCK)
    big = torch.frexp(x.abs().amax(1, keepdim=True))[1] - 1          # 2^big <= the largest < 2^(big + 1)
    scale = torch.ldexp(torch.ones_like(big, dtype=torch.float64), torch.clamp(big, min=32 - 127) - top)
    y = x.abs() / scale
    step = torch.ldexp(torch.ones_like(y), torch.clamp(torch.frexp(y)[1] - 1, min=lowest) - 3)
    return torch.floor(y / step + u.view(-1, BLOCK).double() / 65536) * step * scale * torch.sign(x), step * scale


def _moments(s):
    """The averages in hand in float64."""
    if s["case"]["bits"] == 32:
        return s["m"].double(), s["v"].double()
    m, v = s["m"].long(), s["v"].long()
    out = []
    for code, scale, bias, top in ((m & 127, s["m_scale"], 7, 7), (v, s["v_scale"], 15, 14)):
        e, f = code >> 3, (code & 7).double()
        y = torch.where(e > 0, torch.ldexp(8 + f, e - 3 - bias), torch.ldexp(f, torch.full_like(e, -2 - bias)))
        out.append(torch.ldexp(y, scale.long()[:, None] - 127 - top))
    return (out[0] * (1.0 - 2.0 * (m >> 7).double())).view(-1), out[1].view(-1)


def _adamw_exact(s):
    case, out = s["case"], {}
    g = s["grad"].double()
    if case["clip"]:
        norm = torch.linalg.vector_norm(g)
        out["norm"] = norm
        g = g * min(1.0, 1.0 / (float(norm) + 1e-6))
    t = int(s["step"]) + 1
    out["step"] = torch.tensor(t)
    m, v = _moments(s)
    m, v = torch.lerp(g, m, B1), torch.lerp(g.square(), v, B2)
    p = (s["param"] if s["master"] is None else s["master"]).double()
    rate = torch.full_like(p, LR * DECAY)
    rate[s["split"]:] = 0
    p = p - rate * p - LR * (m / (1 - B1 ** t)) / ((v / (1 - B2 ** t)).sqrt() + ADAM_EPS)
    if case["bits"] == 8:
        u = _random16(m.numel(), s["seed"], t)
        m = _rounded(m, u // 256 + (u % 256) * 256, -6, 7)[0].view(-1)
        r, step = _rounded(v, u, -14, 14)
        v = torch.where((r == 0) & (v.view(-1, BLOCK) > 0), step, r).view(-1)  # no positive average becomes a zero
    out.update(param=p, m=m, v=v)
    if s["master"] is not None:
        out["master"] = p
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        return torch.linalg.vector_norm(s["grad"].double())
    return {"heads": _heads_exact, "adamw": _adamw_exact}[case["op"]](s)

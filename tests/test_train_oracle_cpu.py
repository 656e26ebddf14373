"""The training operators' float64 restatement against its own differences and against autograd, to 64-bit accuracy:
its gradient formulas are written by hand, and the kernels are compared with them."""
import math

import pytest
import torch

from oracle import train_ref as ref

F64 = torch.float64


def attention_case(p):
    g = torch.Generator().manual_seed(7)
    q, do = (torch.randn(2, 19, 6, 8, generator=g, dtype=F64) for _ in range(2))
    k, v = (torch.randn(2, 19, 2, 8, generator=g, dtype=F64) for _ in range(2))
    keep = ref.keep_factor(2 * 6 * 19, 19, p, 3, 4, 5).view(2, 6, 19, 19) if p else None
    return q, k, v, do, keep


@pytest.mark.parametrize("p", [0.0, 0.3])
def test_attention_gradients(p):
    q, k, v, do, keep = attention_case(p)
    pads = [0, 7]
    r = ref.attention(q, k, v, do, pads, 0.4, keep)

    def forward(q, k, v):  # by the definition, on all heads at once
        B, S, Hq, D = q.shape
        R = Hq // k.shape[2]
        s = 0.4 * torch.einsum("bqhd,bkhd->bhqk", q, k.repeat_interleave(R, 2))
        at, pad = torch.arange(S), torch.tensor(pads)
        seen = (at[None, None] <= at[None, :, None]) & (at[None, None] >= pad[:, None, None])
        e = torch.exp(s) * seen[:, None]
        P = e / e.sum(-1, keepdim=True).clamp_min(1e-300)
        return torch.einsum("bhqk,bkhd->bqhd", P if keep is None else P * keep, v.repeat_interleave(R, 2))

    xs = [t.clone().requires_grad_() for t in (q, k, v)]
    out = forward(*xs)
    out.backward(do)
    for name, want in zip(("out", "dq", "dk", "dv"), (out.detach(), *(t.grad for t in xs))):
        assert (r[name][0] - want).abs().max() <= 1e-12 * (1 + want.abs().max()), name
    # And by central differences along the gradient, whose slope is its norm: e^2 of a third derivative, and rounding
    # of 1e-16 / e of sums of some hundreds.
    for i, name in enumerate(("dq", "dk", "dv")):
        grad = r[name][0]
        d, e = grad / grad.norm(), 1e-4
        ends = []
        for sign in (1, -1):
            moved = [q, k, v]
            moved[i] = moved[i] + sign * e * d
            ends.append((ref.attention(*moved, do, pads, 0.4, keep)["out"][0] * do).sum())
        assert abs((ends[0] - ends[1]) / (2 * e) - grad.norm()) <= 1e-6 * grad.norm(), name


@pytest.mark.parametrize("post,gates", [(True, 3), (True, 12), (False, 1), (False, 0)])
def test_residual_norm_gradients(post, gates):
    g = torch.Generator().manual_seed(9)
    M, H, alpha, eps = 12, 10, 0.7, 1e-5

    def rn(*s):
        return torch.randn(*s, generator=g, dtype=F64)

    t = dict(x=rn(M, H), residual=rn(M, H), w_pre=rn(H), w_post=rn(H) if post else None, gate=rn(gates, H) if gates else None)
    dh, dn, keep = rn(M, H), rn(M, H), ref.keep_factor(M, H, 0.3, 1, 2, 3)
    r = ref.residual_norm(t["x"], t["residual"], t["w_pre"], t["w_post"], t["gate"], alpha, eps, keep, dh, dn)
    x = {n: None if v is None else v.clone().requires_grad_() for n, v in t.items()}

    def norm(v, w):
        return v / torch.sqrt(v.pow(2).sum(-1, keepdim=True) / H + eps) * w

    u = norm(x["x"], x["w_post"]) if post else x["x"]
    gate = x["gate"].repeat_interleave(M // gates, 0) if gates else 1.0
    h = x["residual"] + alpha * gate * (u * keep)
    n = norm(h, x["w_pre"])
    ((h * dh).sum() + (n * dn).sum()).backward()
    for name, want in (("h", h.detach()), ("n", n.detach()), ("dx", x["x"].grad), ("dres", x["residual"].grad),
                       ("dpre", x["w_pre"].grad), ("dpost", post and x["w_post"].grad), ("dgate", gates and x["gate"].grad)):
        if r[name] is None:
            assert want is False or want == 0
            continue
        assert (r[name][0] - want).abs().max() <= 1e-12 * (1 + want.abs().max()), name


def test_magnitudes_bound_their_results():
    q, k, v, do, keep = attention_case(0.3)
    for name, (value, size) in ref.attention(q, k, v, do, [0, 7], None, keep).items():
        if not name.endswith("_delta"):
            assert (value.abs() <= size * (1 + 1e-12)).all(), name
    assert math.isclose(ref.keep_factor(1, 8, 0.5, 0, 0, 0).max().item(), 2.0)

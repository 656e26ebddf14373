"""The training attention's gradients away from unit scale, against the float64 restatement.

Bounds are those of tests/test_train_ops_gpu.py without its absolute term for fp16: with u = 2^-11 and A the
absolute terms of a result, u A for the one rounding of P or dS, u |y| for the result's, u of delta's terms
beyond one block of keys, 2^-18 A for the fp32 steps.  What fp16's subnormals may add, by their half steps:
2^-25 for the result itself.  P reaches dv scaled by 2^15 (half step 2^-40 of it), and dS reaches dq and dk
scaled by the power of two that brings c = 2 / (1 - p) max|dO row| max|v row| of the sample and KV head, which
no |dS| exceeds, to 2^14 or more: a half step is at most 2^-39 c there.
"""
import math

import pytest
import torch

from oracle import train_ref as ref
from test_train_ops_gpu import attn_inputs, attn_run, check, no_device_error  # noqa: F401

FP16 = torch.float16
U, SLACK = 2.0 ** -11, 2.0 ** -18


def tolerances(host, dout, pads, p, keep):
    q, k, v = (t.double() for t in host)
    g = dout.double()
    B, S, Hq, D = q.shape
    Hkv = k.shape[2]
    R = Hq // Hkv
    r = ref.attention(q, k, v, g, pads, None, keep)
    tol = {}
    for name in ("dq", "dk", "dv"):
        want, mag = r[name]
        tol[name] = U * 1.01 * (want.abs() + mag) + SLACK * mag + 2.0 ** -25 * 1.01
        if name != "dv":
            off, size = r[name + "_delta"]
            tol[name] += U * 1.01 * off + SLACK * size
    inv = 65536 / (65536 - round(p * 65536))
    for b in range(B):
        lo = min(pads[b], S)
        for h in range(Hkv):
            mine = slice(h * R, (h + 1) * R)
            gg, kk, qq, vv = g[b, lo:, mine], k[b, lo:, h], q[b, lo:, mine], v[b, lo:, h]
            c = 2 * inv * gg.norm(dim=-1).max().item() * vv.norm(dim=-1).max().item() if lo < S else 0.0
            tol["dq"][b, lo:, mine] += 2.0 ** -39 * c / math.sqrt(D) * kk.abs().sum(0)
            tol["dk"][b, lo:, h] += 2.0 ** -39 * c / math.sqrt(D) * qq.abs().sum((0, 1))
            tol["dv"][b, lo:, h] += 2.0 ** -40 * inv * gg.abs().sum((0, 1))
    return r, tol


def run(host, dout, pads, p, rng=(77, 5, 3)):
    B, S, Hq, D = host[0].shape
    keep = ref.keep_factor(B * Hq * S, S, p, *rng).view(B, Hq, S, S) if p > 0 else None
    got, _ = attn_run(tuple(t.cuda() for t in host), dout.cuda(), pads, p, rng)
    r, tol = tolerances(host, dout, pads, p, keep)
    for name, t in zip(("dq", "dk", "dv"), got[1:]):
        check(name, t, r[name][0], tol[name])
    return r


CASES = [
    # B, S, Hq, Hkv, D, pads, p, scale of dout: one block of keys, several, walks that are cut or split
    (2, 40, 4, 2, 64, [0, 7], 0.1, 1e-4),
    (3, 192, 8, 2, 32, [0, 96, 191], 0.0, 1e-4),
    (1, 1000, 4, 2, 64, [0], 0.0, 1e-2),
    (1, 1300, 4, 2, 32, [9], 0.1, 1e-4),
    (2, 1100, 6, 2, 64, [0, 300], 0.2, 1e-4),
    (1, 2500, 2, 2, 64, [0], 0.0, 1e-3),
    (1, 2055, 2, 1, 32, [5], 0.1, 1e-5),
    (40, 130, 6, 2, 64, [(7 * b) % 130 for b in range(40)], 0.1, 1e-3),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"B{c[0]}_S{c[1]}_{c[2]}x{c[3]}_D{c[4]}_p{c[6]}_{c[7]}")
def test_small_fp16_gradients(case):
    B, S, Hq, Hkv, D, pads, p, size = case
    host, dout, _, _ = attn_inputs(B, S, Hq, Hkv, D, FP16, seed=S)
    run(host, (dout.double() * size).to(FP16), pads, p)


@pytest.mark.gpu
def test_fp16_gradients_of_samples_and_heads_of_different_size():
    """Each sample's and KV head's gradients are as exact as if they stood alone."""
    host, dout, _, _ = attn_inputs(3, 700, 4, 2, 64, FP16, seed=31)
    size = torch.tensor([1.0, 1e-2, 1e-4]).view(3, 1, 1, 1) * torch.tensor([1.0, 1.0, 2e-2, 2e-2]).view(1, 1, 4, 1)
    run(host, (dout.double() * size).to(FP16), [0, 3, 130], 0.1)


@pytest.mark.gpu
@pytest.mark.parametrize("S,p", [(50, 0.0), (300, 0.1), (1100, 0.0)])
def test_large_fp16_gradients(S, p):
    """|dS| of up to some 1e5 is no overflow where the gradients themselves fit the type."""
    host, dout, _, _ = attn_inputs(2, S, 4, 2, 64, FP16, seed=S)
    host = ((host[0].double() * 0.3).to(FP16), (host[1].double() * 0.3).to(FP16), (host[2].double() * 100).to(FP16))
    r = run(host, (dout.double() * 250).to(FP16), [0, 9], p)
    assert max(r[n][0].abs().max().item() for n in ("dq", "dk", "dv")) < 60000


@pytest.mark.gpu
def test_fp16_gradients_without_any():
    """All-zero gradients give zeros; a sample that is all padding has no row to take a maximum over."""
    host, dout, _, _ = attn_inputs(2, 90, 4, 2, 32, FP16, seed=1)
    got, _ = attn_run(tuple(t.cuda() for t in host), torch.zeros_like(dout).cuda(), [0, 90])
    assert all((t == 0).all() for t in got[1:])
    run(host, dout, [4, 90], 0.0)


@pytest.mark.gpu
def test_fp16_padding_does_not_set_the_scale():
    """Infinities, NaN and huge values in padded rows change nothing."""
    host, dout, dev, ddev = attn_inputs(2, 300, 4, 2, 64, FP16, seed=8, fused=False)
    ddev = ddev * 1e-3
    want, _ = attn_run(dev, ddev, [0, 70])
    bad = [t.clone() for t in (*dev, ddev)]
    for i, t in enumerate(bad):
        t[1, :70] = (float("inf"), 6e4, float("nan"), 6e4)[i]
    got, _ = attn_run(bad[:3], bad[3], [0, 70])
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.gpu
@pytest.mark.parametrize("R,D,S", [(70, 32, 40), (65, 64, 130), (3, 64, 200)])
def test_heads_do_not_mix(R, D, S):
    """NaN in all of one KV head's rows (its query heads, keys, values and their gradient) leaves the other's results
    as they were, also where the last chunk of 64 query heads is not full."""
    _, _, dev, ddev = attn_inputs(2, S, 2 * R, 2, D, torch.bfloat16, seed=R, fused=False)
    want, _ = attn_run(dev, ddev, [0, 5], 0.1, (5, 6, 7))
    for g in (0, 1):
        bad = [t.clone() for t in (*dev, ddev)]
        for t in bad:
            n = t.shape[2] // 2
            t[:, :, g * n:(g + 1) * n] = float("nan")
        got, _ = attn_run(bad[:3], bad[3], [0, 5], 0.1, (5, 6, 7))
        for w, t in zip(want, got):
            n = t.shape[2] // 2
            keep = slice((1 - g) * n, (2 - g) * n)
            assert torch.equal(w[:, :, keep], t[:, :, keep])


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,Hkv,D,dt", [(1, 1, 64, torch.bfloat16), (4, 2, 32, FP16), (3, 1, 64, torch.bfloat16)])
def test_how_far_values_that_are_not_finite_reach(Hq, Hkv, D, dt):
    """A NaN in k or v: rows more than 190 positions before it keep their results; in q or dout: keys more than 127
    positions behind it.  (fp16 gradients take one scale from a sample's finite values, which the NaN leaves.)"""
    S, at = 700, 411
    _, _, dev, ddev = attn_inputs(1, S, Hq, Hkv, D, dt, seed=9, fused=False)
    want, _ = attn_run(dev, ddev, [3])
    for which in range(4):
        bad = [t.clone() for t in (*dev, ddev)]
        bad[which][:, at] = float("nan")
        got, _ = attn_run(bad[:3], bad[3], [3])
        if which in (1, 2):
            for w, t in zip(want[:2], got[:2]):
                assert torch.isfinite(t[:, :at - 190]).all() and torch.isnan(t[:, at:]).all()
                assert torch.equal(w[:, :at - 190], t[:, :at - 190]) or dt == FP16
        else:
            for w, t in zip(want[2:], got[2:]):
                assert torch.isfinite(t[:, at + 128:]).all()
                assert torch.equal(w[:, at + 128:], t[:, at + 128:]) or dt == FP16


@pytest.mark.gpu
@pytest.mark.parametrize("gate", ["none", "channel", "sample", "token"])
@pytest.mark.parametrize("H,dt", [(264, torch.bfloat16), (130, torch.float32), (64, FP16), (1001, torch.float32)])
def test_residual_norm_drops_whatever_the_value(gate, H, dt):
    """NaN and infinities of x where it is dropped give what zeros there give, in every result and gradient."""
    from test_train_ops_gpu import norm_inputs, norm_run

    B, S = 3, 20
    gates = {"none": 0, "channel": 1, "sample": B, "token": B * S}[gate]
    shape = {"none": None, "channel": (H,), "sample": (B, 1, H), "token": (B, S, H)}[gate]
    host = norm_inputs(B * S, H, dt, False, gates, seed=H)
    rng = (31, 4, 2)
    dropped = ref.keep_factor(B * S, H, 0.3, *rng) == 0
    zero, bad = dict(host), dict(host)
    zero["x"] = host["x"].masked_fill(dropped, 0.0)
    odd = torch.where(torch.arange(H) % 2 == 0, float("nan"), float("inf")).to(dt)
    bad["x"] = torch.where(dropped, odd, host["x"])
    a, b = (norm_run(h, shape, p=0.3, rng=rng, shape=(B, S, H)) for h in (zero, bad))
    for x, y in zip(a, b):
        assert (x is None) == (y is None)
        if x is not None:
            assert torch.isfinite(y).all() and torch.equal(x, y)


@pytest.mark.gpu
def test_status_of_a_device_without_an_index():
    from rl_for_mario_b200.kernels import device_status

    assert device_status(torch.device("cuda")) == 0 and device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("S,D,dt,p", [(20, 32, torch.bfloat16, 0.0), (90, 64, torch.bfloat16, 0.2), (150, 32, FP16, 0.0)])
def test_attention_gradient_along_itself(S, D, dt, p):
    """The slope of the float64 forward pass along each gradient, by central differences: it is the gradient's norm.
    An element off by t moves the kernels' slope along d by t |d|, all of them by |t| |d| = |t| at most (Cauchy and
    Schwarz), t the elementwise bound: a few u of the norm."""
    B, Hq, Hkv, pads, rng = 2, 4, 2, [0, 6], (77, 5, 3)
    host, dout, _, _ = attn_inputs(B, S, Hq, Hkv, D, dt, seed=S)
    keep = ref.keep_factor(B * Hq * S, S, p, *rng).view(B, Hq, S, S) if p > 0 else None
    got, _ = attn_run(tuple(t.cuda() for t in host), dout.cuda(), pads, p, rng)
    r = ref.attention(*host, dout, pads, None, keep)
    u = torch.finfo(dt).eps / 2
    for i, name in enumerate(("dq", "dk", "dv")):
        want, mag = r[name]
        tol = u * 1.01 * (want.abs() + mag) + SLACK * mag + (2.0 ** -22 if dt == FP16 else 0.0)
        if name != "dv":
            tol = tol + u * 1.01 * r[name + "_delta"][0] + SLACK * r[name + "_delta"][1]
        d, e, ends = want / want.norm(), 1e-4, []
        for sign in (1, -1):
            moved = [t.double() for t in host]
            moved[i] = moved[i] + sign * e * d
            ends.append((ref.attention(*moved, dout, pads, None, keep)["out"][0] * dout.double()).sum())
        slope = ((ends[0] - ends[1]) / (2 * e)).item()
        bound = tol.norm().item() + 1e-6 * want.norm().item()
        assert bound < 0.08 * want.norm().item()  # so a gradient wrong by a tenth fails
        assert abs((got[1 + i].double().cpu() * d).sum().item() - slope) <= bound, name


@pytest.mark.gpu
@pytest.mark.parametrize("H", [96, 257, 1001, 4096, 5000])
def test_residual_norm_parts_are_one_wave(H):
    """The backward pass leaves one partial row of each weight's gradient for each block that the GPU holds at a time:
    sixteen warps an SM, a row's ceil(H / 256) warps in blocks of eight or more."""
    from rl_for_mario_b200 import _lib

    sms = torch.cuda.get_device_properties(0).multi_processor_count
    wpr = -(-H // 256)
    block = wpr * max(1, 8 // wpr)
    rows = sms * max(1, 16 // block)
    need = _lib.load().dt_residual_norm_workspace(100000, H, 0, 1)
    assert 0 < need <= 4 * (2 * rows * (-(-H // 4) * 4) + 16)


@pytest.mark.gpu
def test_captured_fp16_backward_scales_by_its_own_gradients():
    """A replay takes the scale of the gradients that stand in its inputs then."""
    from rl_for_mario_b200 import kernels

    _, _, dev, ddev = attn_inputs(2, 300, 4, 2, 64, FP16, seed=12)
    pad = torch.tensor([0, 17], dtype=torch.int32, device="cuda")
    out, lse = kernels.attn_train_forward(*dev, pad)
    d = ddev.clone()
    want = [kernels.attn_train_backward(ddev * s, *dev, out, lse, pad) for s in (1.0, 2.0 ** -12, 8.0)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = kernels.attn_train_backward(d, *dev, out, lse, pad)
    for s, w in zip((1.0, 2.0 ** -12, 8.0), want):
        d.copy_(ddev * s)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, w))

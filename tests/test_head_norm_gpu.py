"""Norms of query and key heads with the rotation in the same pass, and their gradient, against the float64
restatement (oracle/step_ref.py).

Tolerances, elementwise: one rounding of the result, u |y| with u = eps / 2 of its type, and 2^-24 for
each fp32 step on the terms' absolute sum A.  Of a head: 8 products and sums of a lane, 5 shuffles, mean
and eps make 15 steps, halved by the root, rsqrt's 2 ulp 4, and 4 products and sums to a result: under 16
forward.  Backward takes two such sums and twice the products: 64 holds both.  A weight's gradient adds, in
these sizes, the terms of one item of a thread (12 heads at most), 5 shuffles, 8 warps, and the blocks' parts
(592 blocks at most: 19 a lane, then 32), each term off by the 64 of its own: 160.  fp16 numbers under 2^-14 are off by
up to 2^-25.
"""
import pytest
import torch

from oracle import step_ref as ref

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
EPS = 1e-5


@pytest.fixture(autouse=True)
def no_device_error(request):
    yield
    if "gpu" in request.keywords and torch.cuda.is_available():
        from rl_for_mario_b200.kernels import device_status

        torch.cuda.synchronize()
        assert device_status() == 0


def check(name, got, want, mag, steps):
    dt = got.dtype
    tol = torch.finfo(dt).eps / 2 * want.abs() * 1.01 + steps * 2.0 ** -24 * mag + (2.0 ** -25 if dt == FP16 else 0)
    got = got.detach().double().cpu()
    assert got.shape == want.shape, name
    assert torch.isfinite(got).all(), name
    over = ((got - want).abs() - tol).max().item()
    assert over <= 0, f"{name}: {over:.3e} over its bound"


def tables(rows, D, seed=0):
    """Tables whose halves differ, so that a mix-up of the two shows."""
    g = torch.Generator().manual_seed(seed)
    ang = torch.rand(rows, D, generator=g) * 6.2831853
    return ang.cos(), ang.sin()


def make(B, S, Hq, Hkv, D, dt, wdt, seed=0):
    g = torch.Generator().manual_seed(seed)
    qkv = (torch.randn(B, S, Hq + 2 * Hkv, D, generator=g) * torch.randn(B, S, 1, 1, generator=g).exp()).to(dt)
    wq, wk = ((1 + 0.2 * torch.randn(D, generator=g)).to(wdt) for _ in range(2))
    dq, dk = torch.randn(B, S, Hq, D, generator=g).to(dt), torch.randn(B, S, Hkv, D, generator=g).to(dt)
    return qkv, wq, wk, dq, dk


def compare(q, k, wq, wk, cos, sin, pos, dq, dk, got, eps=EPS):
    for n, x, w, d in (("q", q, wq, dq), ("k", k, wk, dk)):
        r = ref.head_norm_rope(x, w, cos, sin, eps, pos, d)
        check(n, got[n], *r["out"], 16)
        check("d" + n, got["d" + n], *r["dx"], 64)
        check("dw" + n, got["dw" + n], *r["dw"], 160)


CASES = [
    # B, S, Hq, Hkv, D, dtype, weights, start
    (1, 1, 1, 1, 2, FP32, FP32, False),
    (1, 3, 8, 2, 32, BF16, BF16, False),
    (2, 5, 3, 1, 6, FP16, FP16, True),
    (3, 7, 4, 4, 8, BF16, FP32, False),
    (2, 33, 5, 5, 42, FP32, FP32, True),
    (5, 3, 6, 2, 16, FP32, FP32, True),
    (4, 189, 8, 2, 32, BF16, FP32, False),
    (1, 255, 12, 4, 64, FP16, FP32, True),
    (3, 64, 2, 1, 66, BF16, BF16, False),
    (2, 65, 3, 3, 128, BF16, BF16, True),
    (3, 17, 4, 1, 130, FP16, FP16, False),
    (2, 31, 2, 2, 254, FP32, FP32, False),
    (7, 11, 2, 1, 256, BF16, BF16, False),
    (3, 21, 3, 2, 48, BF16, BF16, False),   # whole vectors on a group of lanes that it does not fill
    (2, 40, 4, 2, 96, FP16, FP32, True),
    (2, 13, 7, 1, 240, BF16, FP32, False),
    (3, 14, 3, 3, 24, FP32, FP32, True),
    (2, 9, 5, 2, 200, FP32, FP32, False),
    (1, 4, 3, 1, 72, BF16, BF16, False),    # 16-bit heads of an odd number of vectors
    (2, 19, 1, 2, 256, FP32, FP32, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("B,S,Hq,Hkv,D,dt,wdt,start", CASES)
def test_heads_and_gradients(B, S, Hq, Hkv, D, dt, wdt, start):
    from rl_for_mario_b200 import kernels

    qkv, wq, wk, dq, dk = make(B, S, Hq, Hkv, D, dt, wdt)
    rows = S + (40 if start else 0)
    cos, sin = tables(rows, D)
    first = torch.arange(B) * 7 % 41 if start else torch.zeros(B, dtype=torch.long)
    pos = first[:, None] + torch.arange(S)
    dev = qkv.cuda()
    q, k, _ = dev.split([Hq, Hkv, Hkv], 2)
    how = (wq.cuda(), wk.cuda(), EPS, cos.cuda(), sin.cuda(), first.int().cuda() if start else None)
    qo, ko = kernels.head_norm_rope_forward(q, k, *how)
    gq, gk, gwq, gwk = kernels.head_norm_rope_backward(dq.cuda(), dk.cuda(), q, k, *how)
    assert qo.is_contiguous() and gq.is_contiguous() and gwq.dtype == wdt
    hq, hk, _ = qkv.split([Hq, Hkv, Hkv], 2)
    compare(hq, hk, wq, wk, cos, sin, pos, dq, dk, dict(q=qo, k=ko, dq=gq, dk=gk, dwq=gwq, dwk=gwk))
    assert torch.equal(dev.cpu(), qkv)


@pytest.mark.gpu
@pytest.mark.parametrize("D,dt,off", [(32, BF16, 1), (64, FP32, 1), (42, FP16, 1), (64, BF16, 4), (128, FP16, 4), (96, FP32, 4)])
def test_any_strides_and_alignment(D, dt, off):
    """Heads before positions, gaps, an offset of one element or four (16-bit heads on 8-byte boundaries), a table that
    is a slice of a wider one, expanded gradients."""
    from rl_for_mario_b200 import kernels

    B, S, Hq, Hkv = 3, 9, 4, 2
    qkv, wq, wk, dq, dk = make(B, S, Hq, Hkv, D, dt, dt, 3)
    hq, hk, _ = qkv.split([Hq, Hkv, Hkv], 2)
    cos, sin = tables(S, D, 5)
    pos = torch.arange(S).expand(B, S)
    wide = torch.zeros(S, 2 * D + off, device="cuda")
    wide[:, off:D + off], wide[:, D + off:] = cos.cuda(), sin.cuda()
    how = (wq.cuda(), wk.cuda(), EPS, wide[:, off:D + off], wide[:, D + off:])

    def moved(t):
        """The same numbers: off the boundary, [B, H, S, D] in memory with gaps."""
        b, s, n, d = t.shape
        gap = 3 if off == 1 else off
        buf = torch.full((b * n * s * (d + gap) + off,), float("nan"), dtype=t.dtype, device="cuda")
        v = buf[off:].view(b, n, s, d + gap)[..., :d].permute(0, 2, 1, 3)
        v.copy_(t)
        return v

    q, k = moved(hq), moved(hk)
    qo, ko = kernels.head_norm_rope_forward(q, k, *how)
    gq, gk, gwq, gwk = kernels.head_norm_rope_backward(moved(dq), moved(dk), q, k, *how)
    compare(hq, hk, wq, wk, cos, sin, pos, dq, dk, dict(q=qo, k=ko, dq=gq, dk=gk, dwq=gwq, dwk=gwk))
    # One gradient row for every position, last dimension not contiguous.
    one = dq[:1, :1].expand(B, S, Hq, D)
    gq, gk, gwq, gwk = kernels.head_norm_rope_backward(one[:1, :1].cuda().expand(B, S, Hq, D), moved(dk),
                                                       q.transpose(2, 3).contiguous().transpose(2, 3), k, *how)
    compare(hq, hk, wq, wk, cos, sin, pos, one, dk, dict(q=qo, k=ko, dq=gq, dk=gk, dwq=gwq, dwk=gwk))


@pytest.mark.gpu
@pytest.mark.parametrize("D", [32, 42])
def test_gradient_written_over_its_input(D):
    """dq and dk in place of dq_out and dk_out, inside one gradient of q | k | v whose v part stays."""
    from rl_for_mario_b200 import kernels

    B, S, Hq, Hkv = 2, 37, 6, 2
    qkv, wq, wk, dq, dk = make(B, S, Hq, Hkv, D, BF16, BF16, 9)
    cos, sin = tables(S, D)
    dev = qkv.cuda()
    q, k, _ = dev.split([Hq, Hkv, Hkv], 2)
    how = (wq.cuda(), wk.cuda(), EPS, cos.cuda(), sin.cuda())
    want = kernels.head_norm_rope_backward(dq.cuda(), dk.cuda(), q, k, *how)
    g = torch.full_like(dev, 7.0)
    gq, gk, gv = g.split([Hq, Hkv, Hkv], 2)
    gq.copy_(dq), gk.copy_(dk)
    got = kernels.head_norm_rope_backward(gq, gk, q, k, *how, grads=(gq, gk))
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert (gv == 7).all()


@pytest.mark.gpu
def test_many_positions_of_a_thread():
    """More heads than the GPU holds at a time: groups that take several turns, a last one that is not full."""
    from rl_for_mario_b200 import kernels

    B, S, Hq, Hkv, D = 401, 193, 7, 3, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randn(B, S, Hq, D, generator=g, device="cuda").bfloat16()
    k = torch.randn(B, S, Hkv, D, generator=g, device="cuda").bfloat16()
    dq, dk = torch.randn(q.shape, generator=g, device="cuda").bfloat16(), torch.randn(k.shape, generator=g, device="cuda").bfloat16()
    wq, wk = torch.ones(D, device="cuda"), torch.ones(D, device="cuda") * 0.5
    cos, sin = (t.cuda() for t in tables(S, D))
    qo, ko = kernels.head_norm_rope_forward(q, k, wq, wk, EPS, cos, sin)
    gq, gk, gwq, gwk = kernels.head_norm_rope_backward(dq, dk, q, k, wq, wk, EPS, cos, sin)
    again = kernels.head_norm_rope_backward(dq, dk, q, k, wq, wk, EPS, cos, sin)
    for a, b in zip((gq, gk, gwq, gwk), again):
        assert torch.equal(a, b)
    pos = torch.arange(S).expand(B, S)
    for n, x, w, d, o, gx, gw in (("q", q, wq, dq, qo, gq, gwq), ("k", k, wk, dk, ko, gk, gwk)):
        r = ref.head_norm_rope(x.cpu(), w.cpu(), cos.cpu(), sin.cpu(), EPS, pos, d.cpu())
        check(n, o, *r["out"], 16)
        check("d" + n, gx, *r["dx"], 64)
        # 77,393 positions of 7 (3) heads over 207 (88) blocks of 64 groups: 41 terms a thread, one more turn of up to
        # 7, 5 shuffles, 8 warps, 7 parts a lane and 32 lanes: 100, each term off by the 64 of its own.
        check("dw" + n, gw, *r["dw"], 164)


@pytest.mark.gpu
def test_positions_outside_the_tables_and_zero_sizes():
    from rl_for_mario_b200 import kernels

    B, S, D = 3, 4, 32
    q = torch.randn(B, S, 2, D, device="cuda").bfloat16()
    k = torch.randn(B, S, 1, D, device="cuda").bfloat16()
    w = torch.ones(D, device="cuda")
    cos, sin = (t.cuda() for t in tables(10, D))
    start = torch.tensor([0, 8, -1], dtype=torch.int32, device="cuda")
    qo, ko = kernels.head_norm_rope_forward(q, k, w, w, EPS, cos, sin, start)
    torch.cuda.synchronize()
    assert kernels.device_status() != 0 and kernels.device_status() == 0
    good, _ = kernels.head_norm_rope_forward(q[:1], k[:1], w, w, EPS, cos, sin)
    assert torch.equal(qo[0], good[0]) and (qo[1, :2] != 0).any() and (qo[2, 1:] != 0).any()
    assert (qo[1, 2:] == 0).all() and (ko[1, 2:] == 0).all() and (qo[2, 0] == 0).all()
    dq, dk, dwq, dwk = kernels.head_norm_rope_backward(q, k, q, k, w, w, EPS, cos, sin, start)
    torch.cuda.synchronize()
    assert kernels.device_status() != 0
    assert (dq[1, 2:] == 0).all() and torch.isfinite(dwq).all()
    for b, s in ((0, 4), (2, 0)):
        e = torch.empty(b, s, 2, D, device="cuda")
        qo, ko = kernels.head_norm_rope_forward(e, e[:, :, :1], w, w, EPS, cos, sin)
        assert qo.shape == e.shape and ko.shape == (b, s, 1, D)
        out = kernels.head_norm_rope_backward(e, e[:, :, :1], e, e[:, :, :1], w, w, EPS, cos, sin)
        assert (out[2] == 0).all() and (out[3] == 0).all()


@pytest.mark.gpu
def test_values_that_are_not_finite_stay_in_their_head():
    from rl_for_mario_b200 import kernels

    q = torch.randn(2, 3, 4, 32, device="cuda").bfloat16()
    k = torch.randn(2, 3, 2, 32, device="cuda").bfloat16()
    q[1, 1, 2, 5], q[0, 0, 0, 0] = float("nan"), float("inf")
    w = torch.ones(32, device="cuda")
    cos, sin = (t.cuda() for t in tables(3, 32))
    qo, ko = kernels.head_norm_rope_forward(q, k, w, w, EPS, cos, sin)
    bad = ~torch.isfinite(qo).all(-1)
    assert bad[1, 1, 2] and bad[0, 0, 0] and bad.sum() == 2 and torch.isfinite(ko).all()
    # A head of zeros has no direction: zeros, as eps is there.
    q.zero_()
    assert (kernels.head_norm_rope_forward(q, k, w, w, EPS, cos, sin)[0] == 0).all()


@pytest.mark.gpu
def test_another_stream_and_a_graph():
    from rl_for_mario_b200 import kernels

    qkv, wq, wk, dq, dk = (t.cuda() for t in make(4, 50, 8, 2, 32, BF16, FP32))
    q, k, _ = qkv.split([8, 2, 2], 2)
    cos, sin = (t.cuda() for t in tables(60, 32))
    start = torch.zeros(4, dtype=torch.int32, device="cuda")

    def both():
        o = kernels.head_norm_rope_forward(q, k, wq, wk, EPS, cos, sin, start)
        return (*o, *kernels.head_norm_rope_backward(dq, dk, q, k, wq, wk, EPS, cos, sin, start))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = both()
    start.fill_(9)
    qkv.mul_(0.5)
    graph.replay()
    want = both()
    for a, b in zip(captured, want):
        assert torch.equal(a, b)

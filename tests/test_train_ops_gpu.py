"""The training operators' kernels against their float64 restatement (oracle/train_ref.py).

Tolerances are elementwise and follow from where the kernels round.  With
u = eps / 2 of the 16-bit type and A the sum of the absolute terms of a result:
attention rounds P (out, dv) or dS (dq, dk) to the type once, u A, and the
result once, u |y|; where a row's keys span several tiles delta comes from the
stored output, u sum |O| |dO|, which reaches dq and dk through P k and P q.
fp32 steps (products, exp2, sums) add a few 2^-20 of the terms' magnitude: the
product of D terms and its scaling is off by at most (D + 2) 2^-24 of its
absolute sum, exp2 of an argument of up to 32 by 2^-18 relative.  The norm and
dropout operators work in fp32 and round each result once: u |y| + 64 * 2^-24 A
(A the absolute terms; 64 covers the depth of the row sums, 8 per thread + 5
shuffles + up to 32 warps, and of the rows that a thread adds in these sizes).
"""
import pytest
import torch

from oracle import train_ref as ref

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def no_device_error(request):
    """No kernel of a test reports a wait that ran out."""
    yield
    if "gpu" in request.keywords and torch.cuda.is_available():
        from rl_for_mario_b200.kernels import device_status

        torch.cuda.synchronize()
        assert device_status() == 0


def half_eps(dt):
    return torch.finfo(dt).eps / 2


def make_rng(seed, step):
    return torch.tensor([seed, step], dtype=torch.int64, device="cuda")


def check(name, got, want, tol):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, name
    assert torch.isfinite(got).all(), name
    over = (got - want).abs() - tol
    assert over.max().item() <= 0, f"{name}: off by {(got - want).abs().max().item():.3e}, " \
                                   f"{over.max().item():.3e} over its bound"


# ------------------------------------------------------------------------------------- attention
def attn_inputs(B, S, Hq, Hkv, D, dt, seed=0, fused=True):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(B, S, Hq + 2 * Hkv, D, generator=g).to(dt)
    dout = torch.randn(B, S, Hq, D, generator=g).to(dt)
    if fused:
        dev = qkv.cuda()
        q, k, v = dev.split([Hq, Hkv, Hkv], 2)
    else:
        q, k, v = (t.contiguous().cuda() for t in qkv.split([Hq, Hkv, Hkv], 2))
    return qkv.split([Hq, Hkv, Hkv], 2), dout, (q, k, v), dout.cuda()


def attn_check(host, dout, pads, dt, got, p=0.0, rng=(0, 0, 0), scale=None):
    q, k, v = host
    B, S, Hq, D = q.shape
    keep = None
    if p > 0:
        keep = ref.keep_factor(B * Hq * S, S, p, *rng).view(B, Hq, S, S)
    r = ref.attention(q, k, v, dout, pads if pads is not None else [0] * B, scale, keep)
    u, slack = half_eps(dt), 2.0 ** -18
    for name, t in zip(("out", "dq", "dk", "dv"), got):
        want, mag = r[name]
        tol = u * want.abs() * 1.01 + u * mag * 1.01 + slack * mag
        if name in ("dq", "dk"):
            off, size = r[name + "_delta"]
            tol = tol + u * off * 1.01 + slack * size
        if dt == FP16:
            tol = tol + 2.0 ** -24 * 4  # below 2^-14 fp16 steps are 2^-24, in P, dS and the result
        check(name, t, want, tol)


def attn_run(dev, dout, pads, p=0.0, rng=(0, 0, 0), scale=None):
    from rl_for_mario_b200 import kernels

    pad = None if pads is None else torch.tensor(pads, dtype=torch.int32, device="cuda")
    kw = dict(scale=scale, p=p, rng=make_rng(*rng[:2]) if p > 0 else None, site=rng[2])
    out, lse = kernels.attn_train_forward(*dev, pad, **kw)
    return (out, *kernels.attn_train_backward(dout, *dev, out, lse, pad, **kw)), lse


ATTN = [
    # B, S, Hq, Hkv, D, pads, dtype, p
    (1, 1, 8, 2, 32, None, BF16, 0.0),
    (2, 1, 4, 4, 64, [0, 1], FP16, 0.5),
    (1, 3, 8, 2, 32, None, BF16, 0.1),
    (3, 2, 1, 1, 64, [0, 1, 2], BF16, 0.0),
    (2, 63, 4, 2, 32, [0, 17], BF16, 0.1),
    (2, 64, 4, 2, 64, [0, 63], FP16, 0.0),
    (2, 65, 6, 2, 64, [1, 64], BF16, 0.2),
    (4, 192, 8, 2, 32, [0, 96, 191, 192], BF16, 0.1),
    (2, 192, 8, 2, 32, None, FP16, 0.0),
    (2, 191, 8, 1, 32, [0, 33], BF16, 0.1),
    (3, 189, 8, 8, 32, [0, 65, 1000], FP16, 0.3),
    (2, 193, 8, 2, 32, [0, 150], BF16, 0.1),
    (2, 256, 3, 3, 64, [0, 130], FP16, 0.1),
    (1, 257, 12, 4, 64, None, BF16, 0.0),
    (2, 300, 12, 4, 64, [0, 250], BF16, 0.1),
    (1, 520, 7, 1, 64, [77], BF16, 0.1),
    (1, 700, 2, 1, 32, [3], FP16, 0.9),
    (1, 1001, 4, 2, 64, None, FP16, 0.0),
    (1, 1300, 3, 1, 32, [513], BF16, 0.0),
    (1, 70, 70, 1, 32, [5], BF16, 0.1),   # more query heads on a KV head than a tile packs
    (200, 33, 5, 1, 32, "each", BF16, 0.1),  # many short units: a CTA walks several, padding on every residue of 8
    (150, 192, 8, 2, 32, "each", BF16, 0.0),
    (40, 130, 6, 2, 64, "each", FP16, 0.2),
    (1, 2048, 2, 1, 32, [9], BF16, 0.1),  # 64 positions for each of D: the longest whose drop flags are kept
    (1, 2055, 2, 1, 32, [9], BF16, 0.1),
    # Few rows, long walks over the keys, cut into segments: tiles of one segment and of several, padding that
    # leaves fewer of them, packed heads, a row whose last segment lies behind it.
    (1, 1500, 1, 1, 64, None, FP16, 0.2),
    (3, 1100, 3, 1, 64, [0, 517, 1099], BF16, 0.0),
    (2, 2300, 2, 2, 32, [1203, 3], BF16, 0.1),
    (1, 1030, 8, 2, 64, [6], FP16, 0.1),
    (1, 1500, 12, 12, 64, [9], BF16, 0.1),  # tiles of 9 and 17 blocks in segments of 8: a single block is left over
    (1, 1500, 12, 12, 32, [9], FP16, 0.0),
]


def attn_id(c):
    return f"B{c[0]}_S{c[1]}_{c[2]}x{c[3]}_D{c[4]}_{'pad' if c[5] else 'full'}_{str(c[6])[6:]}_p{c[7]}"


@pytest.mark.gpu
@pytest.mark.parametrize("case", ATTN, ids=attn_id)
def test_attention_matches_float64(case):
    B, S, Hq, Hkv, D, pads, dt, p = case
    if pads == "each":
        pads = [(7 * b) % (S + 3) for b in range(B)]
    host, dout, dev, ddev = attn_inputs(B, S, Hq, Hkv, D, dt, seed=S + D)
    rng = (123456789012345, 7, 3)
    got, lse = attn_run(dev, ddev, pads, p, rng)
    attn_check(host, dout, pads, dt, got, p, rng)
    for b, pad in enumerate(pads or []):
        lo = min(pad, S)
        for t in got:
            assert (t[b, :lo] == 0).all()
        assert torch.isinf(lse[b, :, :lo]).all() and torch.isfinite(lse[b, :, lo:]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("D,S", [(32, 100), (64, 100), (64, 260), (32, 260)])
def test_attention_scale_and_separate_tensors(D, S):
    host, dout, dev, ddev = attn_inputs(2, S, 4, 2, D, BF16, seed=5, fused=False)
    got, _ = attn_run(dev, ddev, [0, 40], scale=0.05)
    attn_check(host, dout, [0, 40], BF16, got, scale=0.05)


@pytest.mark.gpu
@pytest.mark.parametrize("D,S,pad", [(32, 192, 70), (64, 300, 70), (32, 300, 64), (64, 40, 39)])
def test_attention_never_reads_behind_the_padding(D, S, pad):
    """NaN and infinities in padded rows of every input change nothing and the padded rows stay zero."""
    _, _, dev, ddev = attn_inputs(2, S, 4, 2, D, BF16, seed=8, fused=False)
    rng = (5, 6, 7)
    want, _ = attn_run(dev, ddev, [0, pad], 0.1, rng)
    bad = [t.clone() for t in (*dev, ddev)]
    for i, t in enumerate(bad):
        t[1, :pad] = float("nan") if i % 2 else float("inf")
    got, _ = attn_run(bad[:3], bad[3], [0, pad], 0.1, rng)
    for w, t in zip(want, got):
        assert torch.equal(w, t)


@pytest.mark.gpu
@pytest.mark.parametrize("D,S", [(32, 192), (64, 300), (32, 300), (64, 128)])
def test_attention_later_positions_do_not_reach_earlier_rows(D, S):
    """Causality, forward and in dq: other keys behind a row leave its results bit for bit."""
    _, _, dev, ddev = attn_inputs(1, S, 4, 2, D, BF16, seed=9, fused=False)
    cut = S - 50
    a, _ = attn_run(dev, ddev, None)
    other = [t.clone() for t in dev]
    for t in other:
        t[:, cut:] = 3.0 * t[:, cut:] + 1.0
    b, _ = attn_run(other, ddev, None)
    assert torch.equal(a[0][:, :cut], b[0][:, :cut]) and torch.equal(a[1][:, :cut], b[1][:, :cut])
    assert not torch.equal(a[0][:, cut:], b[0][:, cut:])


@pytest.mark.gpu
def test_attention_peaked_rows_and_large_scores():
    """Scores of +-60: rows with nearly all weight on one key, no overflow."""
    host, dout, dev, ddev = attn_inputs(2, 150, 4, 2, 64, BF16, seed=3)
    host = tuple((t.float() * (4.0 if i < 2 else 1.0)).to(BF16) for i, t in enumerate(host))
    dev = tuple(t.cuda() for t in host)
    got, _ = attn_run(dev, ddev, [0, 20])
    # exp2's argument reaches 2^7 here: its fp32 rounding is 2^-17 relative, times four for the slack of 2^-18.
    r = ref.attention(*host, dout, [0, 20])
    u = half_eps(BF16)
    for name, t in zip(("out", "dq", "dk", "dv"), got):
        want, mag = r[name]
        tol = u * (want.abs() + mag) * 1.01 + 2.0 ** -16 * mag
        if name in ("dq", "dk"):
            tol = tol + u * r[name + "_delta"][0] * 1.01 + 2.0 ** -16 * r[name + "_delta"][1]
        check(name, t, want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("S,D", [(192, 32), (300, 64), (300, 32)])
def test_attention_is_deterministic_and_keyed(S, D):
    _, _, dev, ddev = attn_inputs(3, S, 8, 2, D, BF16, seed=1)
    a, _ = attn_run(dev, ddev, [0, 5, 100], 0.1, (1, 2, 3))
    b, _ = attn_run(dev, ddev, [0, 5, 100], 0.1, (1, 2, 3))
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    for other in ((2, 2, 3), (1, 3, 3), (1, 2, 4), (1 + (1 << 40), 2, 3)):
        c, _ = attn_run(dev, ddev, [0, 5, 100], 0.1, other)
        assert not torch.equal(a[0], c[0])


@pytest.mark.gpu
def test_attention_gradient_against_differences():
    """d(sum out * dout) / dx by central differences of the float64 restatement's forward."""
    host, dout, dev, ddev = attn_inputs(1, 20, 2, 1, 32, BF16, seed=2)
    got, _ = attn_run(dev, ddev, [4])

    def loss(q, k, v):
        return (ref.attention(q, k, v, dout, [4])["out"][0] * dout.double()).sum().item()

    g = torch.Generator().manual_seed(4)
    for which in range(3):
        base = [t.double() for t in host]
        direction = torch.randn(base[which].shape, generator=g, dtype=torch.float64)
        e = 1e-4
        hi, lo = list(base), list(base)
        hi[which], lo[which] = base[which] + e * direction, base[which] - e * direction
        want = (loss(*hi) - loss(*lo)) / (2 * e)
        grad = got[1 + which].double().cpu()
        # Each element is off by up to 2 u (|y| + A), A some |y| in size: their errors in one direction add up to at
        # most sum |direction| * 4 u |grad|-sized terms; the difference quotient itself is off by O(e^2).
        bound = 4 * half_eps(BF16) * (direction.abs() * (grad.abs() + grad.abs().mean())).sum().item() + 1e-5
        assert abs((grad * direction).sum().item() - want) <= bound


@pytest.mark.gpu
def test_attention_scratch_is_checked_on_the_host():
    """A shape whose walks over keys are cut needs scratch in both directions: too little, none or a misaligned
    one is refused before anything is launched, and a shape that needs none takes a null pointer."""
    from rl_for_mario_b200 import _lib

    lib = _lib.load()
    S, D = 1500, 64
    t = torch.zeros(1, S, 1, D, dtype=BF16, device="cuda")
    lse = torch.zeros(1, 1, S, device="cuda")
    need = lib.dt_attn_train_forward_workspace(1, S, 1, 1, D)
    assert need > 0 and lib.dt_attn_train_forward_workspace(64, 192, 8, 2, 32) == 0
    ws = torch.zeros(need + 16, dtype=torch.uint8, device="cuda")
    out = torch.zeros_like(t)

    def forward(pointer, size):
        q = t.data_ptr()
        return lib.dt_attn_train_forward(q, q, q, out.data_ptr(), lse.data_ptr(), None, 1, S, 1, 1, D,
                                         *(S * D, D, D) * 4, pointer, size, 0.0, 0.0, None, 0, 0, None)

    assert forward(None, need) != 0 and forward(ws.data_ptr(), need - 4) != 0 and forward(ws.data_ptr() + 4, need) != 0
    assert forward(ws.data_ptr(), need) == 0
    plain, drop = (lib.dt_attn_train_workspace(1, S, 1, 1, D, has) for has in (0, 1))
    assert 0 < plain < drop
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_cut_attention_on_two_streams_and_in_a_graph():
    """Calls whose walks are cut, at once on two streams and replayed from a graph: each has scratch of its own."""
    _, _, dev, ddev = attn_inputs(1, 1500, 2, 2, 64, BF16, seed=21)
    _, _, dev2, ddev2 = attn_inputs(2, 1100, 3, 1, 64, BF16, seed=22)
    want = attn_run(dev, ddev, [9], 0.1, (3, 4, 5))[0]
    want2 = attn_run(dev2, ddev2, [0, 77], 0.0)[0]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    runs = []
    for _ in range(3):
        with torch.cuda.stream(streams[0]):
            a = attn_run(dev, ddev, [9], 0.1, (3, 4, 5))[0]
        with torch.cuda.stream(streams[1]):
            b = attn_run(dev2, ddev2, [0, 77], 0.0)[0]
        runs.append((a, b))
    torch.cuda.synchronize()
    for a, b in runs:
        assert all(torch.equal(x, y) for x, y in zip(want, a)) and all(torch.equal(x, y) for x, y in zip(want2, b))

    from rl_for_mario_b200 import kernels

    pad, rng = torch.tensor([9], dtype=torch.int32, device="cuda"), make_rng(3, 4)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = kernels.attn_train_forward(*dev, pad, p=0.1, rng=rng, site=5)
        grads = kernels.attn_train_backward(ddev, *dev, out, lse, pad, p=0.1, rng=rng, site=5)
    for t in (out, lse, *grads):
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(want, (out, *grads)))


@pytest.mark.gpu
def test_attention_two_streams_and_a_captured_graph():
    from rl_for_mario_b200 import kernels

    _, _, dev, ddev = attn_inputs(2, 192, 8, 2, 32, BF16, seed=6)
    _, _, dev2, ddev2 = attn_inputs(2, 300, 4, 2, 64, FP16, seed=7)
    a, _ = attn_run(dev, ddev, None, 0.1, (3, 4, 5))
    b, _ = attn_run(dev2, ddev2, None, 0.1, (3, 4, 5))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    res = []
    for _ in range(4):
        for st, (x, d) in zip(streams, ((dev, ddev), (dev2, ddev2))):
            with torch.cuda.stream(st):
                res.append(attn_run(x, d, None, 0.1, (3, 4, 5))[0])
    torch.cuda.synchronize()
    for i, r in enumerate(res):
        assert all(torch.equal(x, y) for x, y in zip(r, (a, b)[i % 2]))

    rng = make_rng(3, 4)

    def step():
        out, lse = kernels.attn_train_forward(*dev, p=0.1, rng=rng, site=5)
        return (out, *kernels.attn_train_backward(ddev, *dev, out, lse, p=0.1, rng=rng, site=5))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(outs, a))
    rng[1] += 1  # a replay reads the step that stands there
    graph.replay()
    torch.cuda.synchronize()
    want, _ = attn_run(dev, ddev, None, 0.1, (3, 5, 5))
    assert all(torch.equal(x, y) for x, y in zip(outs, want))
    assert not torch.equal(outs[0], a[0])


@pytest.mark.gpu
def test_attention_backward_into_one_gradient_and_odd_strides():
    from rl_for_mario_b200 import kernels

    _, _, dev, ddev = attn_inputs(2, 70, 4, 2, 32, BF16, seed=12)
    want, _ = attn_run(dev, ddev, [0, 9])
    pad = torch.tensor([0, 9], device="cuda")  # int64 is taken too
    out, lse = kernels.attn_train_forward(*dev, pad)
    whole = torch.full((2, 70, 8, 32), 7.0, dtype=BF16, device="cuda")
    parts = (whole[:, :, :4], whole[:, :, 4:6], whole[:, :, 6:])
    kernels.attn_train_backward(ddev, *dev, out, lse, pad, grads=parts)
    for w, t in zip(want[1:], parts):
        assert torch.equal(w, t)
    # Inputs whose rows the kernels cannot read in place: odd strides, an expanded gradient, [B, H, S, D] order.
    q = torch.zeros(2, 70, 4, 33, dtype=BF16, device="cuda")[..., :32].copy_(dev[0])
    k = dev[1].transpose(1, 2).contiguous().transpose(1, 2)
    ones = torch.ones((), dtype=BF16, device="cuda").expand(2, 70, 4, 32)
    a = kernels.attn_train_backward(ones, q, k, dev[2], out, lse, pad)
    b = kernels.attn_train_backward(ones.contiguous(), *dev, out, lse, pad)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


# -------------------------------------------------------------------------------- residual + norms
def norm_inputs(M, H, dt, post, gates, seed=0, residual=True):
    g = torch.Generator().manual_seed(seed)

    def rn(*s, m=1.0, c=0.0):
        return (torch.randn(*s, generator=g) * m + c).to(dt)

    return dict(x=rn(M, H), residual=rn(M, H, m=2.0) if residual else None, w_pre=rn(H, m=0.1, c=1.0),
                w_post=rn(H, m=0.1, c=1.0) if post else None, gate=rn(gates, H, m=0.3, c=0.5) if gates else None,
                dh=rn(M, H), dn=rn(M, H))


def norm_check(host, dev_out, dt, alpha, eps, p, rng, dh=True, dn=True):
    M, H = host["x"].shape
    keep = ref.keep_factor(M, H, p, *rng)
    r = ref.residual_norm(host["x"], host["residual"], host["w_pre"], host["w_post"], host["gate"], alpha, eps, keep,
                          host["dh"] if dh else None, host["dn"] if dn else None)
    u = half_eps(dt)
    for name, got in zip(("h", "n", "dx", "dres", "dpre", "dpost", "dgate"), dev_out):
        if r[name] is None:
            assert got is None
            continue
        want, mag = r[name]
        tiny = 2.0 ** -24 if dt == FP16 else 0.0  # the step of fp16's subnormals
        check(name, got.reshape(want.shape), want, u * want.abs() * 1.001 + 64 * 2.0 ** -24 * mag + tiny)


def norm_run(host, gate_shape=None, alpha=0.7, eps=1e-5, p=0.0, rng=(0, 0, 0), dh=True, dn=True, shape=None):
    from rl_for_mario_b200 import kernels

    dev = {k: None if v is None else v.cuda() for k, v in host.items()}
    if shape is not None:
        for k in ("x", "residual", "dh", "dn"):
            dev[k] = None if dev[k] is None else dev[k].view(shape)
    gate = dev["gate"]
    if gate is not None:
        gate = gate.view(gate_shape)
    kw = dict(post_weight=dev["w_post"], gate=gate, alpha=alpha, p=p, rng=make_rng(*rng[:2]) if p > 0 else None,
              site=rng[2])
    h, n, stats = kernels.residual_norm_forward(dev["x"], dev["residual"], dev["w_pre"], eps, **kw)
    g = kernels.residual_norm_backward(dev["dh"] if dh else None, dev["dn"] if dn else None, dev["x"],
                                       dev["residual"], dev["w_pre"], stats, **kw)
    return (h, n, *g)


NORM = [
    # shape, dtype, post, gate, p, residual
    ((1, 1, 8), BF16, False, "none", 0.0, True),
    ((1, 3, 256), BF16, False, "none", 0.1, True),
    ((2, 5, 1), FP32, True, "channel", 0.0, True),
    ((3, 7, 13), FP32, True, "sample", 0.3, True),
    ((3, 64, 256), FP16, True, "sample", 0.1, True),
    ((5, 129, 257), BF16, True, "channel", 0.1, False),
    ((2, 200, 768), BF16, True, "token", 0.1, True),
    ((4, 33, 1001), FP32, True, "sample", 0.1, True),
    ((4, 33, 1001), FP16, False, "token", 0.0, True),
    ((2, 100, 2048), FP32, False, "channel", 0.5, True),
    ((2, 30, 2056), BF16, True, "channel", 0.1, True),
    ((1, 9, 4099), BF16, True, "sample", 0.1, True),
    ((1, 5, 8192), FP32, True, "channel", 0.1, True),
    ((500, 1, 264), BF16, False, "sample", 0.0, True),
    ((700, 3, 64), BF16, True, "sample", 0.2, True),
    ((9, 192, 256), BF16, False, "none", 0.1, True),
    ((2, 700, 5000), BF16, True, "channel", 0.1, True),  # rows of more than 16 warps, several for each block
    ((3, 300, 8192), FP16, True, "sample", 0.0, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", NORM, ids=lambda c: "x".join(map(str, c[0])) + f"_{str(c[1])[6:]}_{c[2]}_{c[3]}_p{c[4]}")
def test_residual_norm_matches_float64(case):
    (B, S, H), dt, post, gate, p, residual = case
    gates = {"none": 0, "channel": 1, "sample": B, "token": B * S}[gate]
    gshape = {"none": None, "channel": (H,), "sample": (B, 1, H), "token": (B, S, H)}[gate]
    host = norm_inputs(B * S, H, dt, post, gates, seed=H, residual=residual)
    rng = (99, 1 << 20, 2)
    got = norm_run(host, gshape, p=p, rng=rng, shape=(B, S, H))
    norm_check(host, got, dt, 0.7, 1e-5, p, rng)


@pytest.mark.gpu
@pytest.mark.parametrize("dh,dn", [(True, False), (False, True)])
def test_residual_norm_with_one_gradient(dh, dn):
    host = norm_inputs(70, 96, FP32, True, 1, seed=4)
    got = norm_run(host, (96,), p=0.1, rng=(1, 2, 3), dh=dh, dn=dn)
    norm_check(host, got, FP32, 0.7, 1e-5, 0.1, (1, 2, 3), dh=dh, dn=dn)


@pytest.mark.gpu
def test_residual_norm_strided_rows_and_repeatability():
    from rl_for_mario_b200 import kernels

    host = norm_inputs(300, 264, BF16, True, 1, seed=6)
    a = norm_run(host, (264,), p=0.1, rng=(1, 2, 3))
    b = norm_run(host, (264,), p=0.1, rng=(1, 2, 3))
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    wide = torch.zeros(300, 531, dtype=BF16, device="cuda")
    x = wide[:, 3:267].copy_(host["x"].cuda())  # rows on odd boundaries
    h, n, _ = kernels.residual_norm_forward(x, host["residual"].cuda(), host["w_pre"].cuda(), 1e-5,
                                            post_weight=host["w_post"].cuda(), gate=host["gate"].cuda().view(264),
                                            alpha=0.7, p=0.1, rng=make_rng(1, 2), site=3)
    # Another order of the row sums: results agree to their rounding.
    norm_check(host, (h, n), BF16, 0.7, 1e-5, 0.1, (1, 2, 3))


@pytest.mark.gpu
def test_residual_norm_against_differences():
    host = norm_inputs(6, 40, FP32, True, 2, seed=7)
    rng = (5, 5, 5)
    got = norm_run(host, (2, 1, 40), p=0.2, rng=rng, shape=(2, 3, 40))
    keep = ref.keep_factor(6, 40, 0.2, *rng)

    def loss(**over):
        t = {**host, **over}
        r = ref.residual_norm(t["x"], t["residual"], t["w_pre"], t["w_post"], t["gate"], 0.7, 1e-5, keep, None, None)
        return ((r["h"][0] * host["dh"].double()).sum() + (r["n"][0] * host["dn"].double()).sum()).item()

    g = torch.Generator().manual_seed(1)
    for name, grad in zip(("x", "residual", "w_pre", "w_post", "gate"), got[2:]):
        d = torch.randn(host[name].shape, generator=g, dtype=torch.float64)
        e = 1e-5
        want = (loss(**{name: host[name].double() + e * d}) - loss(**{name: host[name].double() - e * d})) / (2 * e)
        have = (grad.double().cpu().view(d.shape) * d).sum().item()
        # fp32 rounding of each gradient element (64 * 2^-24 of terms a few times its size), differences O(e^2)
        assert abs(have - want) <= 1e-4 * (grad.double().cpu().view(d.shape) * d).abs().sum().item() + 1e-6


# ---------------------------------------------------------------------------------------- dropout
DROP = [
    ((1, 1), BF16, 0.5, False), ((1, 7), FP32, 0.1, True), ((3, 8), FP16, 0.1, False), ((5, 1001), FP32, 0.25, True),
    ((192, 256), BF16, 0.1, True), ((2, 3, 5, 40), FP16, 0.9, True), ((4097, 24), BF16, 0.0, True),
    ((129, 2049), BF16, 0.1, False), ((1000, 520), FP32, 0.001, False),
    # Odd widths: rows that begin at every place of 16 bytes, one column more or less than a warp's.
    ((70, 247), BF16, 0.2, True), ((70, 249), FP16, 0.2, False), ((33, 1001), FP16, 0.1, True),
    ((40, 63), BF16, 0.5, True), ((40, 65), BF16, 0.5, True), ((500, 243), FP32, 0.3, False), ((20, 4093), FP32, 0.1, True),
    ((3, 30011), BF16, 0.0, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("shape,dt,p,residual", DROP, ids=lambda v: str(v).replace(" ", ""))
def test_dropout_matches_float64(shape, dt, p, residual):
    from rl_for_mario_b200 import kernels

    g = torch.Generator().manual_seed(3)
    x, r, dy = (torch.randn(*shape, generator=g).to(dt) for _ in range(3))
    rng = (1 << 50, 11, 8)
    keep = ref.keep_factor(x.numel() // shape[-1], shape[-1], p, *rng).view(shape)
    y = kernels.dropout_forward(x.cuda(), p, make_rng(*rng[:2]), site=8, residual=r.cuda() if residual else None)
    dx = kernels.dropout_backward(dy.cuda(), p, make_rng(*rng[:2]), site=8)
    u = half_eps(dt)
    want = x.double() * keep + (r.double() if residual else 0.0)
    mag = (x.double() * keep).abs() + (r.double().abs() if residual else 0.0)
    tiny = 2.0 ** -24 if dt == FP16 else 0.0
    check("y", y, want, u * want.abs() * 1.001 + 2.0 ** -22 * mag + tiny)
    want = dy.double() * keep
    check("dx", dx, want, u * want.abs() * 1.001 + 2.0 ** -22 * want.abs() + tiny)
    if p > 0:
        assert torch.equal(dx.cpu() == 0, (keep == 0) | (dy == 0))


@pytest.mark.gpu
def test_dropout_drops_whatever_the_value_and_takes_strides():
    from rl_for_mario_b200 import kernels

    rng = make_rng(4, 5)
    x = torch.full((64, 130), float("nan"), device="cuda")
    keep = ref.keep_factor(64, 130, 0.5, 4, 5, 0)
    y = kernels.dropout_forward(x, 0.5, rng)
    assert torch.equal(torch.isnan(y).cpu(), keep > 0) and (y[(keep == 0).cuda()] == 0).all()
    base = torch.randn(64, 200, device="cuda", dtype=BF16)
    for view in (base[:, 8:136], base[:, 3:131], base.t()[:128].t(), base[::2, :128], base[:1, :128].expand(64, 128)):
        assert torch.equal(kernels.dropout_forward(view, 0.3, rng), kernels.dropout_forward(view.contiguous(), 0.3, rng))


@pytest.mark.gpu
def test_dropout_rate():
    """The share kept of 2^24 elements is within six standard deviations of 1 - p."""
    from rl_for_mario_b200 import kernels

    n = 1 << 24
    for p in (0.1, 0.5):
        y = kernels.dropout_forward(torch.ones(n // 512, 512, device="cuda"), p, make_rng(17, 23), site=1)
        q = round(p * 65536) / 65536
        assert abs((y == 0).double().mean().item() - q) <= 6 * (q * (1 - q) / n) ** 0.5

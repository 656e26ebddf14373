"""Refusals of the head norms that need no GPU."""
import pytest
import torch


def test_head_norm_entry_points_refuse_bad_arguments():
    from rl_for_mario_b200 import _lib

    lib = _lib.load()
    a, INV, UNS = 4096, _lib.DT_ERR_INVALID, _lib.DT_ERR_UNSUPPORTED

    def fwd(q=a, out=a, cos=a, cos_stride=32, rows=8, start=None, B=1, S=8, Hq=4, Hkv=2, D=32, strides=(8,) * 12,
            w=a, w32=0, eps=1e-5, dtype=0):
        st = (_lib._L * len(strides))(*strides) if strides else None
        return lib.dt_head_norm_rope_forward(q, a, w, a, out, a, cos, a, cos_stride, rows, start, B, S, Hq, Hkv, D, st,
                                             w32, eps, dtype, None)

    for kw, code in ((dict(q=None), INV), (dict(out=None), INV), (dict(w=None), INV), (dict(cos=None), INV),
                     (dict(strides=None), INV), (dict(B=0), INV), (dict(S=0), INV), (dict(Hkv=0), INV),
                     (dict(D=33), UNS), (dict(D=0), UNS), (dict(D=258), UNS), (dict(dtype=3), UNS),
                     (dict(q=a + 1), INV), (dict(w=a + 2, w32=1), INV), (dict(cos=a + 2), INV),
                     (dict(start=a + 2), INV), (dict(rows=7), INV), (dict(rows=0, start=a), INV),
                     (dict(cos_stride=31), INV), (dict(strides=(-8,) + (8,) * 11), INV), (dict(eps=-1.0), INV),
                     (dict(eps=float("nan")), INV), (dict(B=1 << 20, S=1 << 10, start=a), UNS)):
        assert fwd(**kw) == code, kw

    def bwd(g=a, dw=a, ws=a, size=1 << 30):
        st = (_lib._L * 18)(*(8,) * 18)
        return lib.dt_head_norm_rope_backward(g, a, a, a, a, a, a, a, dw, a, a, a, 32, 8, None, ws, size, 1, 8, 4, 2, 32,
                                              st, 0, 1e-5, 0, None)

    assert bwd(g=None) == INV and bwd(dw=None) == INV
    assert lib.dt_head_norm_rope_workspace(1, 8, 4, 2, 31) < 0 and lib.dt_head_norm_rope_workspace(0, 8, 4, 2, 32) < 0


@pytest.mark.parametrize("D", [2, 6, 32])
def test_head_norm_gradient_against_differences(D):
    """The oracle's gradient against central differences of its forward pass: with h = 2^-17 they are off by h^2 times
    a third derivative (sizes here: some tens) and by 2^-52 / h of the sum."""
    from oracle import step_ref as ref

    g = torch.Generator().manual_seed(D)
    x, w = torch.randn(2, 3, 2, D, generator=g, dtype=torch.float64), 1 + 0.3 * torch.randn(D, generator=g, dtype=torch.float64)
    cos, sin, d = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((5, D), (5, D), x.shape))
    pos = torch.tensor([[0, 3, 4], [1, 2, 2]])
    r = ref.head_norm_rope(x, w, cos, sin, 1e-2, pos, d)
    h = 2.0 ** -17

    def value(x, w):
        return (ref.head_norm_rope(x, w, cos, sin, 1e-2, pos)["out"][0] * d).sum().item()

    for n, t in (("dx", x), ("dw", w)):
        for i in range(0, t.numel(), max(1, t.numel() // 40)):
            e = torch.zeros_like(t).view(-1)
            e[i] = h
            e = e.view_as(t)
            args = [(x + e, w), (x - e, w)] if n == "dx" else [(x, w + e), (x, w - e)]
            diff = (value(*args[0]) - value(*args[1])) / (2 * h)
            assert abs(diff - r[n][0].view(-1)[i].item()) < 1e-6 * (1 + abs(diff)), (n, i)


def test_head_norm_wrapper_checks():
    from rl_for_mario_b200 import kernels as K

    q, k, w = torch.zeros(2, 4, 4, 32), torch.zeros(2, 4, 2, 32), torch.ones(32)
    t = torch.zeros(4, 32)
    with pytest.raises(ValueError, match="CUDA"):
        K.head_norm_rope_forward(q, k, w, w, 1e-5, t, t)
    with pytest.raises(ValueError, match="CUDA"):
        K.head_norm_rope_backward(q, k, q, k, w, w, 1e-5, t, t)
    ok = (q, k, w, w, 1e-5, t, t, None)
    assert K._check_head_norm(*ok)[3:] == (2, 4, 4, 2, 32)

    def refused(kind, match, **kw):
        names = ("q", "k", "q_weight", "k_weight", "eps", "cos", "sin", "start_pos")
        args = dict(zip(names, ok))
        args.update(kw)
        with pytest.raises(kind, match=match):
            K._check_head_norm(**args)

    refused(ValueError, "takes q", q=q[0])
    refused(ValueError, "match", k=k[:1])
    refused(TypeError, "dtype", k=k.half())
    refused(TypeError, "dtype", q=q.double(), k=k.double())
    refused(ValueError, "even", q=torch.zeros(2, 4, 4, 31), k=torch.zeros(2, 4, 2, 31))
    refused(ValueError, "even", q=torch.zeros(2, 4, 1, 258), k=torch.zeros(2, 4, 1, 258))
    refused(ValueError, "one head", k=k[:, :, :0])
    refused(ValueError, "2.31", q=torch.empty(2, 4, 4, 32).expand(2, 4, 4, 32).as_strided((2 ** 16, 2 ** 15, 4, 32), (0, 0, 0, 1)),
            k=torch.empty(32).as_strided((2 ** 16, 2 ** 15, 2, 32), (0, 0, 0, 1)))
    refused(ValueError, "contiguous", q_weight=torch.ones(64)[::2])
    refused(ValueError, "contiguous", k_weight=torch.ones(31))
    refused(TypeError, "fp32", q_weight=w.half())
    refused(TypeError, "fp32", q_weight=w.half(), k_weight=w.half())
    refused(ValueError, "eps", eps=-1.0)
    refused(ValueError, "eps", eps=float("nan"))
    refused(ValueError, "eps", eps=1e39)
    refused(ValueError, "tables", cos=t[:3], sin=t[:3])
    refused(ValueError, "tables", cos=t[:, :16], sin=t[:, :16])
    refused(ValueError, "tables", sin=torch.zeros(5, 32))
    refused(ValueError, "start_pos", start_pos=torch.zeros(3, dtype=torch.int32))
    assert K._check_head_norm(*ok[:7], torch.zeros(2, dtype=torch.int64))[2].dtype == torch.int32


def test_step_entry_points_refuse_bad_arguments():
    import math

    from rl_for_mario_b200 import _lib
    from rl_for_mario_b200.optim import _GROUP

    lib = _lib.load()
    a, INV, UNS = 4096, _lib.DT_ERR_INVALID, _lib.DT_ERR_UNSUPPORTED
    L, I = _lib._L, _lib._I

    def arrays(p, g, n, kind):
        return (L * 1)(p), (L * 1)(g), (L * 1)(n), (I * 1)(kind)

    def norm(g=a, n=8, kind=0, count=1, out=a, ws=a, size=1 << 20):
        _, gs, ns, ks = arrays(0, g, n, kind)
        return lib.dt_grad_norm(count, gs, ns, ks, out, ws, size, None)

    for kw, code in ((dict(count=0), INV), (dict(out=None), INV), (dict(ws=None), INV), (dict(size=7), INV),
                     (dict(g=a + 1), INV), (dict(g=a + 2, kind=2), INV), (dict(n=-1), INV), (dict(n=1 << 40), INV),
                     (dict(kind=3), UNS), (dict(kind=256), INV), (dict(kind=-256), INV), (dict(out=a + 2), INV)):
        assert norm(**kw) == code, kw
    assert lib.dt_grad_norm_workspace(0) < 0

    def step(count=1, p=a, g=a, n=8, kind=0, ngroups=1, group=(1e-3, 0.9, 0.999, 1e-8, 0.0, 0), bits=32, m=a, s=None,
             master=None, state=a, ticket=a, max_norm=0.0, norm=None, ws=None, size=0):
        ps, gs, ns, ks = arrays(p, g, n, kind)
        return lib.dt_adamw_step(count, ps, gs, ns, ks, ngroups, _GROUP.pack(*group), bits, m, a, s, s, master, state,
                                 ticket, max_norm, norm, ws, size, None)

    bad = [dict(count=0), dict(p=0), dict(p=a + 1), dict(g=a + 1), dict(n=-1), dict(kind=256), dict(m=None), dict(m=a + 8),
           dict(bits=8), dict(master=a + 4), dict(state=None), dict(state=a + 4), dict(ticket=None), dict(ticket=a + 2),
           dict(max_norm=1.0), dict(max_norm=1.0, norm=a), dict(max_norm=math.nan), dict(max_norm=1e-60, norm=a, ws=a),
           dict(max_norm=1.0, norm=a, ws=a + 8, size=1 << 20)]
    for i, wrong in enumerate((-1.0, 1.0, 1.0, 0.0, -1.0)):  # lr, betas, eps, decay
        group = [1e-3, 0.9, 0.999, 1e-8, 0.0, 0]
        for w in (wrong, math.nan, math.inf):
            group[i] = w
            bad.append(dict(group=tuple(group)))
    bad += [dict(group=(1e-3, 0.9, 0.999, eps, 0.0, 0)) for eps in (1e-40, 1e39, -1e-8)]
    bad.append(dict(group=(1e-3, 0.9, 0.999, 1e-8, 0.0, a + 1)))
    for kw in bad:
        assert step(**kw) == INV, kw
    for kw in (dict(kind=3), dict(ngroups=0), dict(ngroups=17), dict(bits=16)):
        assert step(**kw) == UNS, kw
    assert lib.dt_adamw_moments(a, a, a, a, 0, a, a, None) == INV
    assert lib.dt_adamw_moments(a, a, None, a, 1, a, a, None) == INV
    assert lib.dt_adamw_moments(a, a, a, a, 1, a + 8, a, None) == INV


def test_optimizer_refuses_cpu_tensors():
    from rl_for_mario_b200 import optim

    with pytest.raises(ValueError, match="CUDA"):
        optim.AdamW([torch.nn.Parameter(torch.zeros(3))])
    with pytest.raises(ValueError, match="CUDA"):
        optim.grad_norm([torch.zeros(3)])
    assert optim._dense(torch.zeros(3, 4, 5).permute(2, 0, 1)) and optim._dense(torch.zeros(1, 5)[:, :5])
    assert not optim._dense(torch.zeros(4, 4)[:, :3]) and not optim._dense(torch.zeros(1).expand(3))
    assert optim._dense(torch.zeros(0, 3)) and optim._dense(torch.zeros(()))


def test_rounding_at_random_of_the_restatement():
    """The 8-bit form as the oracle states it: every code decodes to a number that is stored as itself whatever its
    word, two neighbours come in the part's proportion, scales are powers of two from the block's largest."""
    import numpy as np

    from oracle import step_ref as ref

    for kind, codes in ((ref.FIRST, np.arange(0, 120)), (ref.SECOND, np.arange(0, 240))):
        block = np.zeros(256, np.uint8)
        block[:len(codes)] = codes
        block[255] = codes[-1]  # of the top binade: the block's scale is its own
        for scale in (32, 100, 127, 254):
            x = ref.decode(block, np.array([scale]), kind)
            assert np.isfinite(x).all() and (np.diff(x[:len(codes)]) > 0).all()
            assert np.array_equal(x.astype(np.float32), torch.from_numpy(x).bfloat16().float().numpy())
            for word in (0, 65535):
                back, e = ref.encode(x, np.full(256, word), kind)
                assert np.array_equal(back, block) and e[0] == scale
    x = np.zeros(256, np.float32)
    x[0], x[1:] = 1.0, 0.3
    up = [ref.encode(x, np.full(256, w), ref.SECOND)[0][1] for w in range(0, 65536, 64)]
    low = min(up)
    a, b = (float(ref.decode(np.full(256, c, np.uint8), np.array([127]), ref.SECOND)[0]) for c in (low, low + 1))
    share = (0.3 - a) / (b - a)
    assert a < 0.3 < b and abs(np.mean([u != low for u in up]) - share) < 2 / 1024


def test_head_norms_of_a_swapped_module():
    from types import SimpleNamespace

    from rl_for_mario_b200.attention import FastDTAttention, swap_attention

    def config(**kw):
        return SimpleNamespace(hidden_size=64, num_attention_heads=2, num_key_value_heads=1, dropout=0.0, **kw)

    class Reference(torch.nn.Module):
        def __init__(self):
            super().__init__()
            for n, k in (("q", 64), ("k", 32), ("v", 32), ("o", 64)):
                setattr(self, n + "_proj", torch.nn.Linear(64, k, bias=False))

    class Block(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.self_attn = Reference()

    block, ref = Block(), None
    ref = block.self_attn
    assert swap_attention(block, config(qk_norm=True, rms_norm_eps=1e-6)) == 1
    m = block.self_attn
    assert torch.equal(m.k_proj.weight, ref.k_proj.weight) and (m.q_norm.weight == 1).all() and m.k_norm.eps == 1e-6
    assert {"q_norm.weight", "k_norm.weight"} <= set(m.state_dict())
    again = FastDTAttention.from_reference(m, config(qk_norm=True))
    assert again.k_norm.eps == 1e-5
    plain = FastDTAttention(config())
    assert set(plain.state_dict()) == {f"{n}_proj.weight" for n in "qkvo"} and plain._head_norms(torch.float32) is None
    with pytest.raises(RuntimeError):
        FastDTAttention.from_reference(m, config())

"""Norms of query and key heads where the framework uses them: the attention module in prefill, cached decode and
training, the whole model, and a training step of it that ends in AdamW.

With u = eps / 2 of the compute type a module's output passes six roundings (projection, head norm, scores' weights,
attention, output projection, and the value's projection), its gradients as many again: results are held to 8 u and
20 u of their norm, which a missing or wrong term exceeds by far; fp32 modules to 64 * 2^-24 (sums of 128 terms).
"""
import math
from types import SimpleNamespace

import pytest
import torch

EPS = 1e-5
pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_device_error():
    yield
    from rl_for_mario_b200.kernels import device_status

    torch.cuda.synchronize()
    assert device_status() == 0


def module(dtype, hidden=128, heads=4, kv_heads=2, dropout=0.0, seed=0):
    from rl_for_mario_b200.attention import FastDTAttention

    torch.manual_seed(seed)
    cfg = SimpleNamespace(hidden_size=hidden, num_attention_heads=heads, num_key_value_heads=kv_heads, dropout=dropout,
                          flash_attn=True, qk_norm=True, rms_norm_eps=EPS)
    m = FastDTAttention(cfg)
    with torch.no_grad():
        for w in (m.q_norm.weight, m.k_norm.weight):
            w.add_(0.3 * torch.randn_like(w))
    return m.cuda().to(dtype)


def tables(S, D):
    from rl_for_mario_b200.dt_model import rope_tables

    return tuple(t.cuda() for t in rope_tables(D, S, 1e4))


def module64(m, x, pads, P):
    """The module in float64; rows before a sample's padding give zeros."""
    B, S, H = x.shape
    Hq, Hkv, D = m.n_local_heads, m.n_local_kv_heads, m.head_dim
    cos, sin = (t.double().cpu()[:, None] for t in tables(S, D))

    def head(t, w):
        t = t * (t.square().mean(-1, keepdim=True) + EPS).rsqrt() * w
        return t * cos + torch.cat((-t[..., D // 2:], t[..., :D // 2]), -1) * sin

    q = head((x @ P["q_proj.weight"].T).view(B, S, Hq, D), P["q_norm.weight"])
    k = head((x @ P["k_proj.weight"].T).view(B, S, Hkv, D), P["k_norm.weight"]).repeat_interleave(Hq // Hkv, 2)
    v = (x @ P["v_proj.weight"].T).view(B, S, Hkv, D).repeat_interleave(Hq // Hkv, 2)
    at = torch.arange(S)
    alive = at[None] >= torch.tensor(pads)[:, None]
    seen = ((at[None] <= at[:, None])[None] & alive[:, None]) | ~alive[:, :, None]
    s = torch.einsum("bqhd,bkhd->bhqk", q, k) / math.sqrt(D)
    a = torch.einsum("bhqk,bkhd->bqhd", torch.softmax(s.masked_fill(~seen[:, None], -math.inf), -1), v)
    return (a * alive[:, :, None, None]).reshape(B, S, -1) @ P["o_proj.weight"].T


def params64(m):
    return {n: t.detach().double().cpu().requires_grad_() for n, t in m.named_parameters()}


def close(name, got, want, bound):
    got = got.detach().double().cpu()
    assert torch.isfinite(got).all(), name
    off = ((got - want).norm() / want.norm()).item()
    assert off <= bound, f"{name}: {off:.3e}"


def unit(dtype):
    return torch.finfo(dtype).eps / 2


@pytest.mark.parametrize("hidden,heads,kv_heads", [(128, 4, 2), (256, 4, 1)], ids=["d32", "d64"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_prefill_and_cached_decode(dtype, hidden, heads, kv_heads):
    from rl_for_mario_b200.cache import PagedKVCache

    m = module(dtype, hidden, heads, kv_heads).eval()
    B, S = 3, 27
    x = torch.randn(B, S, hidden, device="cuda").to(dtype)
    cos, sin = tables(S, m.head_dim)
    P = params64(m)
    bound = 64 * 2.0 ** -24 if dtype == torch.float32 else 8 * unit(dtype)
    want = module64(m, x.double().cpu(), [0] * B, P).detach()
    with torch.no_grad():
        out, _ = m(x, (cos, sin))
        close("prefill", out, want, bound)
        layer = PagedKVCache(1, B, kv_heads, m.head_dim, S, 8, dtype)[0]
        first, past = m(x[:, :10], (cos[:10], sin[:10]), past_key_value=layer, use_cache=True)
        parts, dense = [first], None
        dense = m(x[:, :10], (cos[:10], sin[:10]), use_cache=True)[1]
        tuples = [first]
        for s in range(10, S):
            pe = (cos[s:s + 1], sin[s:s + 1])
            o, past = m(x[:, s:s + 1], pe, past_key_value=layer, use_cache=True)
            parts.append(o)
            o, dense = m(x[:, s:s + 1], pe, past_key_value=dense, use_cache=True)
            tuples.append(o)
        close("paged", torch.cat(parts, 1), want, bound)
        close("dense", torch.cat(tuples, 1), want, bound)


@pytest.mark.parametrize("hidden,heads,kv_heads", [(128, 4, 2), (256, 4, 4)], ids=["d32", "d64"])
@pytest.mark.parametrize("how", ["fp16", "autocast", "compute_dtype"])
def test_training_gradients(how, hidden, heads, kv_heads):
    dtype = torch.float16 if how == "fp16" else torch.float32
    m = module(dtype, hidden, heads, kv_heads).train().fuse_training()
    if how == "compute_dtype":
        m.compute_dtype = torch.float16
    pads, B, S = [0, 5, 19], 3, 33
    g = torch.Generator().manual_seed(2)
    x = torch.randn(B, S, hidden, generator=g).to(dtype).cuda().requires_grad_()
    cot = torch.randn(B, S, hidden, generator=g)
    mask = (torch.arange(S)[None] >= torch.tensor(pads)[:, None])
    with torch.autocast("cuda", torch.float16, enabled=how == "autocast"):
        out, _ = m(x, tables(S, m.head_dim), attention_mask=mask.float().cuda())
    out.backward(cot.to(out.dtype).cuda())
    P = params64(m)
    x64 = x.detach().double().cpu().requires_grad_()
    want = module64(m, x64, pads, P)
    want.backward(cot.to(out.dtype).double())
    close("out", out, want.detach(), 8 * 2.0 ** -11)
    close("dx", x.grad, x64.grad, 20 * 2.0 ** -11)
    for n, t in m.named_parameters():
        assert t.grad.dtype == t.dtype
        close(n, t.grad, P[n].grad, 20 * 2.0 ** -11)


def model(dtype, **kw):
    from rl_for_mario_b200.dt_model import DTConfig, MarioDT

    torch.manual_seed(0)
    cfg = DTConfig(hidden_size=128, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, context_len=8,
                   qk_norm=True, **kw)
    return MarioDT(cfg).cuda().to(dtype)


def batch(m, B=3, T=5, seed=1):
    g = torch.Generator().manual_seed(seed)
    c = m.config
    d = dict(states=torch.randint(0, 256, (B, T, *c.state_shape), generator=g, dtype=torch.uint8),
             actions=torch.randint(0, c.act_dim, (B, T), generator=g), returns_to_go=torch.rand(B, T, generator=g),
             timesteps=torch.arange(T).expand(B, T))
    return {k: v.cuda() for k, v in d.items()}


def test_fused_blocks_agree_and_the_names_stand():
    from rl_for_mario_b200.dt_model import DTConfig

    m = model(torch.float16, dropout=0.0).eval()
    names = {n for n, _ in m.named_parameters() if ".q_norm." in n or ".k_norm." in n}
    assert names == {f"model.layers.{i}.self_attn.{n}_norm.weight" for i in range(2) for n in "qk"}
    b = batch(m)
    with torch.no_grad():
        a = m(**b).action_logits
        m.fuse_norms()
        # Two blocks of some ten roundings each, taken at other places.
        close("fused", m(**b).action_logits, a.double().cpu(), 40 * 2.0 ** -11)
        m.reference_rounding()
        with pytest.raises(ValueError, match="rope_rounding"):
            m(**b)
    old = SimpleNamespace(**{n: getattr(m.config, n) for n in DTConfig.__dataclass_fields__ if n != "qk_norm"})
    assert DTConfig.from_reference(old).qk_norm is False and DTConfig.from_reference(m.config).qk_norm is True


@pytest.mark.parametrize("bits", [8, 32])
def test_training_step_of_a_model_and_its_capture(bits):
    """Loss, gradients, clipped step: eager, then the whole step as one graph."""
    m = model(torch.bfloat16, dropout=0.1).train().fuse_training(seed=5)
    opt = m.adamw(lr=1e-3, weight_decay=0.1, state_bits=bits, master=True, max_norm=1.0, seed=9)
    assert [len(g["params"]) for g in opt.param_groups] == [sum(p.dim() > 1 for p in m.parameters()),
                                                            sum(p.dim() < 2 for p in m.parameters())]
    b = batch(m)

    def step():
        m(**b).loss.backward()
        opt.step()
        opt.zero_grad(set_to_none=True)

    start = {n: p.detach().clone() for n, p in m.named_parameters()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert int(opt.steps()) == 2 and math.isfinite(opt.norm.item())
    moved = 0
    for n, p in m.named_parameters():
        assert torch.isfinite(p).all(), n
        moved += not torch.equal(p, start[n])
    assert moved > 20
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m(**b).loss.backward()
        opt.step()
        opt.zero_grad(set_to_none=True)
    before = opt.master.clone()
    for t in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert int(opt.steps()) == 3 + t and math.isfinite(opt.norm.item())
        assert torch.isfinite(opt.master).all() and not torch.equal(opt.master, before)
        before = opt.master.clone()


def test_attention_with_head_norms_against_its_parts():
    from rl_for_mario_b200 import training

    B, S, Hq, Hkv, D = 2, 40, 6, 2, 32
    g = torch.Generator(device="cuda").manual_seed(3)
    cos, sin = tables(S, D)
    leaves = []
    for _ in range(2):
        g.manual_seed(3)
        leaves.append([torch.randn(B, S, Hq + 2 * Hkv, D, generator=g, device="cuda").bfloat16().requires_grad_(),
                       (1 + 0.1 * torch.randn(D, generator=g, device="cuda")).requires_grad_(),
                       (1 + 0.1 * torch.randn(D, generator=g, device="cuda")).requires_grad_()])
    pad = torch.tensor([0, 7], dtype=torch.int32, device="cuda")
    rng = torch.tensor([3, 4], device="cuda")
    one = training.attention_qk_norm(leaves[0][0], Hq, Hkv, *leaves[0][1:], EPS, cos, sin, pad, p=0.2, rng=rng, site=6)
    q, k, v = leaves[1][0].split([Hq, Hkv, Hkv], 2)
    q, k = training.head_norm_rope(q, k, *leaves[1][1:], EPS, cos, sin)
    two = training.attention(q, k, v, pad, p=0.2, rng=rng, site=6)
    assert torch.equal(one, two)
    d = torch.randn(one.shape, generator=g, device="cuda").bfloat16()
    one.backward(d), two.backward(d)
    for a, b in zip(*leaves):
        assert torch.equal(a.grad, b.grad)
    with pytest.raises(ValueError, match="qkv"):
        training.attention_qk_norm(leaves[0][0], Hq, 1, *leaves[0][1:], EPS, cos, sin)

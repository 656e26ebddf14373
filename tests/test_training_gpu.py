"""The training operators together, as a model uses them: a whole forward and backward pass of the
decoder against a float64 restatement with the same dropout masks, the drop-in module, capture of a
training step, and what fuse_training() leaves alone."""
import math

import pytest
import torch
import torch.nn.functional as F

from oracle import train_ref as ref

EPS = 1e-5


@pytest.fixture(autouse=True)
def no_device_error(request):
    """No kernel of a test reports a wait that ran out."""
    yield
    if "gpu" in request.keywords and torch.cuda.is_available():
        from rl_for_mario_b200.kernels import device_status

        torch.cuda.synchronize()
        assert device_status() == 0


def small_model(dtype, dropout=0.1, hidden=128, heads=4, kv_heads=2, layers=2, context=8, seed=0):
    from rl_for_mario_b200.dt_model import DTConfig, MarioDT

    torch.manual_seed(seed)
    cfg = DTConfig(hidden_size=hidden, num_hidden_layers=layers, num_attention_heads=heads,
                   num_key_value_heads=kv_heads, context_len=context, dropout=dropout)
    m = MarioDT(cfg)
    with torch.no_grad():
        for n, t in m.named_parameters():
            if "norm" in n:
                t.add_(0.1 * torch.randn_like(t))
    return m.cuda().to(dtype)


def norm64(x, w):
    return x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt() * w


def decoder64(model, tokens, pads, seed, step):
    """embed_norm, blocks and final norm in float64 with the masks of (seed, step); autograd gives the gradients."""
    cfg, bb = model.config, model.model
    P = {n: t.detach().double().cpu().requires_grad_() for n, t in bb.named_parameters()}
    B, S, H = tokens.shape
    Hq, Hkv = cfg.num_attention_heads, cfg.num_key_value_heads
    D, R = H // Hq, Hq // Hkv
    p = cfg.dropout
    x = tokens.detach().double().cpu().requires_grad_()

    def drop(t, site):
        return t * ref.keep_factor(B * S, H, p, seed, step, site).view(B, S, H)

    h = drop(norm64(x, P["embed_norm.weight"]), 0)
    cos, sin = (t[:S, None].double().cpu() for t in (bb.freqs_cos, bb.freqs_sin))

    def rot(t):
        return t * cos + torch.cat((-t[..., D // 2:], t[..., :D // 2]), -1) * sin

    at = torch.arange(S)
    seen = (at[None] <= at[:, None])[None] & (at[None, None] >= torch.tensor(pads)[:, None, None])
    alive = (at[None] >= torch.tensor(pads)[:, None]).double()
    for i in range(cfg.num_hidden_layers):
        w = {k[len(f"layers.{i}."):]: v for k, v in P.items() if k.startswith(f"layers.{i}.")}
        n = norm64(h, w["input_layernorm.weight"])
        q = rot((n @ w["self_attn.q_proj.weight"].T).view(B, S, Hq, D))
        k = rot((n @ w["self_attn.k_proj.weight"].T).view(B, S, Hkv, D)).repeat_interleave(R, 2)
        v = (n @ w["self_attn.v_proj.weight"].T).view(B, S, Hkv, D).repeat_interleave(R, 2)
        s = torch.einsum("bqhd,bkhd->bhqk", q, k) / math.sqrt(D)
        s = s.masked_fill(~(seen | (alive == 0)[:, :, None])[:, None], -math.inf)  # empty rows made harmless ...
        keep = ref.keep_factor(B * Hq * S, S, p, seed, step, 1 + 3 * i).view(B, Hq, S, S)
        a = torch.einsum("bhqk,bkhd->bqhd", torch.softmax(s, -1) * keep, v) * alive[:, :, None, None]  # ... and zero
        h = h + drop(a.reshape(B, S, H) @ w["self_attn.o_proj.weight"].T, 2 + 3 * i)
        n = norm64(h, w["post_attention_layernorm.weight"])
        f = F.silu(n @ w["mlp.gate_proj.weight"].T) * (n @ w["mlp.up_proj.weight"].T)
        h = h + drop(f @ w["mlp.down_proj.weight"].T, 3 + 3 * i)
    return x, P, norm64(h, P["norm.weight"])


@pytest.mark.gpu
@pytest.mark.parametrize("hidden,heads,kv_heads,dropout,pads", [
    (128, 4, 2, 0.1, [0, 9, 24]), (128, 4, 2, 0.0, [0, 3, 21]), (256, 4, 1, 0.2, [0, 0, 12])],
    ids=["d32", "d32_p0", "d64"])
def test_decoder_step_matches_float64(hidden, heads, kv_heads, dropout, pads):
    """fp16, u = 2^-11.  A value or gradient passes some 14 roundings a block forward and as many back, 70 in
    all with the embedding and the final norm; each moves a result by at most u of its size (the norms keep every
    stage's scale at 1), so a result's error is at most 70 u = 3.4 % of its norm.  A missing or wrong term of any
    operator is of the result's own size."""
    model = small_model(torch.float16, dropout, hidden, heads, kv_heads).train().fuse_training(seed=77)
    g = torch.Generator().manual_seed(1)
    B, S = 3, 24
    tokens = torch.randn(B, S, hidden, generator=g).half()
    cot = torch.randn(B, S, hidden, generator=g).half()
    for b, pad in enumerate(pads):
        cot[b, :pad] = 0
    x = tokens.cuda().requires_grad_()
    out, _ = model.model.run_training(x, torch.tensor(pads, dtype=torch.int32, device="cuda"))
    out = out.view(B, S, hidden)
    out.backward(cot.cuda())
    x64, P, want = decoder64(model, tokens, pads, 77, 0)
    want.backward(cot.double())
    bound = 70 * 2.0 ** -11
    alive = (torch.arange(S)[None] >= torch.tensor(pads)[:, None])[..., None]

    def close(name, got, exp):
        got = got.double().cpu()
        assert torch.isfinite(got).all(), name
        assert (got - exp).norm() <= bound * exp.norm(), f"{name}: {((got - exp).norm() / exp.norm()).item():.3e}"

    close("out", out.detach() * alive.cuda(), want.detach() * alive)
    close("dx", x.grad, x64.grad)
    n = 0
    for name, t in model.model.named_parameters():
        if name.startswith(("layers", "norm", "embed_norm")):
            close(name, t.grad, P[name].grad)
            n += 1
    assert n == 2 * 9 + 2


def batch(model, B=3, T=5, seed=3, pads=None):
    g = torch.Generator().manual_seed(seed)
    c = model.config
    mask = torch.ones(B, T)
    for b, pad in enumerate(pads or []):
        mask[b, :pad] = 0
    d = dict(states=torch.randint(0, 256, (B, T, *c.state_shape), generator=g, dtype=torch.uint8),
             actions=torch.randint(0, c.act_dim, (B, T), generator=g), returns_to_go=torch.rand(B, T, generator=g),
             timesteps=torch.arange(T).expand(B, T).contiguous(), attention_mask=mask)
    return {k: v.cuda() for k, v in d.items()}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_model_step_reaches_every_parameter(dtype):
    model = small_model(dtype).train().fuse_training(seed=5)
    data = batch(model, pads=[0, 2, 4])
    targets = data["actions"].masked_fill(data["attention_mask"] == 0, -100)
    model(**data, action_targets=targets).loss.backward()
    for n, t in model.named_parameters():
        if n.startswith("value_head"):
            continue  # the action loss does not use it
        assert t.grad is not None and torch.isfinite(t.grad).all() and (t.grad != 0).any(), n
    assert model.model.dropout_state().state_dict() == {"seed": 5, "step": 1}
    first = {n: t.grad.clone() for n, t in model.named_parameters() if t.grad is not None}

    def again(step):
        model.zero_grad()
        model.model.dropout_state().load_state_dict({"seed": 5, "step": step})
        model(**data, action_targets=targets).loss.backward()
        return [t.grad for n, t in model.named_parameters() if n in first and "layers" in n]

    was = [first[n] for n in first if "layers" in n]
    assert all(torch.equal(a, b) for a, b in zip(again(0), was))
    assert not all(torch.equal(a, b) for a, b in zip(again(1), was))


@pytest.mark.gpu
def test_the_generator_moves_with_its_model():
    model = small_model(torch.float16, 0.1, 128, 4, 2).train().fuse_training(seed=11)
    attn = model.model.layers[0].self_attn
    for owner in (model.model, attn):
        for _ in range(2):
            owner.dropout_state().draw()
    model.cpu()
    for owner in (model.model, attn):
        assert owner.dropout_state().state_dict() == {"seed": 11, "step": 2}
        assert owner.dropout_state().state.device.type == "cpu"
    model.cuda()
    for owner in (model.model, attn):
        assert owner.dropout_state().draw().tolist() == [11, 2] and owner.dropout_state().state.is_cuda


@pytest.mark.gpu
def test_every_place_drops_at_its_own_rate():
    """The embedding's, the attention's and the MLP's rate are read apart: with only one of them above zero the
    result still depends on the generator's step, and with none it does not."""
    x = torch.randn(2, 24, 128, generator=torch.Generator().manual_seed(2)).half().cuda()

    def twice(model):
        return [model.model.run_training(x)[0] for _ in range(2)]

    for place in (0, 1, 2, None):
        model = small_model(torch.float16, 0.0, 128, 4, 2).train().fuse_training(seed=5)
        if place == 0:
            model.model.dropout.p = 0.3
        for layer in model.model.layers:
            if place == 1:
                layer.self_attn.dropout = 0.3
            if place == 2:
                layer.mlp.dropout.p = 0.3
        a, b = twice(model)
        assert torch.equal(a, b) == (place is None)
        a, b = twice(model.eval())
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_inference_is_left_alone():
    """Without autograd a model gives the same bits with and without fuse_training(); with autograd and no dropout
    the training form agrees with it to bf16 rounding."""
    model = small_model(torch.bfloat16).eval()
    data = batch(model)
    with torch.no_grad():
        a = model(**data).action_logits
    model.fuse_training(seed=1)
    with torch.no_grad():
        b = model(**data).action_logits
    assert torch.equal(a, b)
    c = model(**data).action_logits
    assert c.requires_grad
    # Two evaluations of one network, each off by at most 40 roundings of u = 2^-8 (a forward pass of two blocks
    # and the encoder), relative to the logits' norm.
    assert (c.detach().float() - a.float()).norm() <= 2 * 40 * 2.0 ** -8 * a.float().norm()
    assert model.model.dropout_state().state_dict()["step"] == 0  # eval mode drops nothing
    model.fuse_training(False)
    assert not model.model.train_form and not model.model.layers[0].self_attn.train_form


@pytest.mark.gpu
def test_drop_in_module_trains_inside_a_plain_block():
    from rl_for_mario_b200.attention import FastDTAttention
    from rl_for_mario_b200.dt_model import DTConfig, rope_tables

    cfg = DTConfig(hidden_size=128, num_attention_heads=4, num_key_value_heads=2, context_len=16, dropout=0.25)
    for dtype, compute in ((torch.bfloat16, None), (torch.float32, torch.bfloat16)):
        torch.manual_seed(0)
        m = FastDTAttention(cfg, compute_dtype=compute).cuda().to(dtype).train().fuse_training(seed=9, site=4)
        x = torch.randn(2, 30, 128, device="cuda").to(dtype).requires_grad_()
        pe = tuple(t.cuda() for t in rope_tables(32, 30, 1e4))
        mask = torch.ones(2, 30, device="cuda")
        mask[1, :7] = 0
        y, past = m(x, pe, attention_mask=mask)
        assert past is None and y.dtype == dtype
        y.float().sum().backward()
        assert all(t.grad is not None and torch.isfinite(t.grad).all() for t in m.parameters())
        # The output's own dropout: site + 1 of the step that this call drew.
        keep = ref.keep_factor(60, 128, 0.25, 9, 0, 5).view(2, 30, 128)
        assert torch.equal((y != 0).cpu(), (keep > 0) & (mask[..., None] > 0).cpu())
        assert (x.grad[1, :7] == 0).all()
    with pytest.raises(TypeError, match="training form"):
        FastDTAttention(cfg).cuda().fuse_training()(x.float(), pe)


@pytest.mark.gpu
def test_captured_training_step_replays_with_new_masks():
    """Forward and backward captured into a graph, while an eager graph of the same leaves is alive is never made:
    the gradients are taken with torch.autograd.grad inside the capture."""
    model = small_model(torch.bfloat16, layers=1).train().fuse_training(seed=3)
    g = torch.Generator().manual_seed(1)
    tokens = torch.randn(2, 24, 128, generator=g).bfloat16().cuda()
    cot = torch.randn(2, 8, 3, 128, generator=g).bfloat16().cuda()
    params = [t for n, t in model.model.named_parameters() if "layers" in n]

    def step():
        out, _ = model.model.run_training(tokens)
        return (out, *torch.autograd.grad(out, params, cot))

    def eager(at):
        model.model.dropout_state().load_state_dict({"seed": 3, "step": at})
        return [t.detach().clone() for t in step()]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [eager(0), eager(1)]
        model.model.dropout_state().load_state_dict({"seed": 3, "step": 0})
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for w in want:
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, w))
    assert model.model.dropout_state().state_dict()["step"] == 2


@pytest.mark.gpu
def test_backward_after_the_generator_moved_on():
    """A backward pass uses the masks of its own forward pass, and a generator changed in place under saved
    tensors is refused by autograd."""
    from rl_for_mario_b200 import training

    st = training.DropoutState(11)
    x = torch.randn(64, 128, device="cuda", requires_grad=True)
    a = training.dropout(x, 0.5, st.draw(), 2)
    b = training.dropout(x, 0.5, st.draw(), 2)
    (ga,), (gb,) = torch.autograd.grad(a.sum(), x), torch.autograd.grad(b.sum(), x)
    assert torch.equal(ga != 0, a != 0) and torch.equal(gb != 0, b != 0) and not torch.equal(ga, gb)
    c = training.dropout(x, 0.5, st.state, 2)
    st.draw()
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(c.sum(), x)


@pytest.mark.gpu
def test_autograd_functions_against_each_other():
    """The packed attention equals the one on three tensors; unused outputs and inputs without gradients."""
    from rl_for_mario_b200 import training

    g = torch.Generator().manual_seed(2)
    qkv = torch.randn(2, 33, 8, 32, generator=g).bfloat16().cuda().requires_grad_()
    q, k, v = (t.detach().contiguous().requires_grad_() for t in qkv.split([4, 2, 2], 2))
    rng = training.DropoutState(1).draw()
    a = training.attention_qkv(qkv, 4, 2, p=0.1, rng=rng, site=6)
    b = training.attention(q, k, v, p=0.1, rng=rng, site=6)
    assert torch.equal(a, b)
    a.sum().backward()
    b.sum().backward()
    assert torch.equal(qkv.grad, torch.cat((q.grad, k.grad, v.grad), 2))
    with pytest.raises(ValueError, match="qkv"):
        training.attention_qkv(qkv, 4, 4)

    x, w = torch.randn(5, 40, device="cuda", requires_grad=True), torch.ones(40, device="cuda", requires_grad=True)
    r = torch.randn(5, 40, device="cuda")
    h, n = training.residual_norm(x, r, w, EPS)
    (gx,) = torch.autograd.grad(h.sum(), x, retain_graph=True)
    assert torch.equal(gx, torch.ones_like(x))
    n.sum().backward()
    x2, w2 = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    norm64(x2 + r.double(), w2).sum().backward()
    for got, want in ((x.grad, x2.grad), (w.grad, w2.grad)):
        # fp32 rounding of 40-term sums of terms of order 1
        assert (got.double() - want).abs().max() <= 64 * 2.0 ** -24 * 10


@pytest.mark.gpu
@pytest.mark.parametrize("D,dt", [(32, torch.bfloat16), (64, torch.float16)])
def test_qkv_rope_gradient_matches_float64(D, dt):
    from rl_for_mario_b200 import training
    from rl_for_mario_b200.dt_model import rope_tables

    g = torch.Generator().manual_seed(D)
    B, S, K, Hq, Hkv = 2, 21, 128, 4, 2
    N = (Hq + 2 * Hkv) * D
    x = torch.randn(B, S, K, generator=g).to(dt)
    w = (torch.randn(N, K, generator=g) / math.sqrt(K)).to(dt)
    dy = torch.randn(B, S, N, generator=g).to(dt)
    cos, sin = rope_tables(D, S, 1e4)
    xd, wd = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    y = training.qkv_rope(xd, wd, cos.cuda(), sin.cuda(), (Hq + Hkv) * D, D)
    keep = dy.cuda()
    y.backward(keep)
    assert torch.equal(keep.cpu(), dy)  # the caller's gradient is not rotated in place
    x64, w64 = x.double().requires_grad_(), w.double().requires_grad_()
    t = (x64 @ w64.T).view(B, S, Hq + 2 * Hkv, D)
    c, s = cos[:, None].double(), sin[:, None].double()
    r = t * c + torch.cat((-t[..., D // 2:], t[..., :D // 2]), -1) * s
    y64 = torch.cat((r[:, :, :Hq + Hkv], t[:, :, Hq + Hkv:]), 2).view(B, S, N)
    y64.backward(dy.double())
    u = torch.finfo(dt).eps / 2
    # The rotated gradient is rounded once and the product once: u (|y| + sum |terms|), with a rotated pair at most
    # |a| + |b| of its two gradients; fp32 sums of N (or B S) terms add N 2^-24 of the terms.
    ga = (dy.double().abs().view(B, S, -1, D) + dy.double().abs().view(B, S, -1, D).roll(D // 2, -1)).view(B * S, N)
    for got, want, mag in ((xd.grad, x64.grad, (ga @ w.double().abs()).view(B, S, K)),
                           (wd.grad, w64.grad, ga.T @ x.double().abs().view(-1, K))):
        tol = u * (want.abs() + mag) * 1.01 + N * 2.0 ** -24 * mag + 2.0 ** -23
        assert ((got.double().cpu() - want).abs() <= tol).all()

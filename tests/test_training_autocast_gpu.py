"""Training under autocast over fp32 weights, as the reference's trainer runs it."""
import math

import pytest
import torch

from oracle import train_ref as ref
from test_training_gpu import batch, decoder64, no_device_error, small_model  # noqa: F401

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def close(name, got, want, bound):
    got = got.double().cpu()
    assert torch.isfinite(got).all(), name
    assert (got - want).norm() <= bound * want.norm(), f"{name}: {((got - want).norm() / want.norm()).item():.3e}"


@pytest.mark.gpu
@pytest.mark.parametrize("ac", [BF16, FP16])
@pytest.mark.parametrize("hidden,heads,kv_heads,p", [(128, 4, 2, 0.2), (256, 4, 1, 0.0), (120, 3, 1, 0.1)],
                         ids=["d32", "d64_p0", "d40_refused"])
def test_drop_in_module_under_autocast(ac, hidden, heads, kv_heads, p):
    """A module with fp32 weights inside a plain fp32 block.  With u the half step of autocast's type, a result passes
    at most 24 roundings (inputs, weights, products, P, the output and their gradients), each u of its size: 24 u
    of its norm.  A missing term is of the result's own size."""
    from rl_for_mario_b200.attention import FastDTAttention
    from rl_for_mario_b200.dt_model import DTConfig, rope_tables

    D = hidden // heads
    cfg = DTConfig(hidden_size=hidden, num_attention_heads=heads, num_key_value_heads=kv_heads, context_len=16, dropout=p)
    torch.manual_seed(0)
    m = FastDTAttention(cfg).cuda().train().fuse_training(seed=9, site=4)
    B, S, pads = 2, 30, [0, 7]
    g = torch.Generator().manual_seed(3)
    x = torch.randn(B, S, hidden, generator=g)
    cot = torch.randn(B, S, hidden, generator=g).to(ac)
    cos, sin = rope_tables(D, S, 1e4)
    mask = torch.ones(B, S)
    mask[1, :7] = 0
    xd = x.cuda().requires_grad_()
    with torch.autocast("cuda", ac):
        if D not in (32, 64):
            with pytest.raises(ValueError, match="head_dim"):
                m(xd, (cos.cuda(), sin.cuda()), attention_mask=mask.cuda())
            return
        y, past = m(xd, (cos.cuda(), sin.cuda()), attention_mask=mask.cuda())
    assert past is None and y.dtype == ac
    y.backward(cot.cuda())

    P = {n: t.detach().double().cpu().requires_grad_() for n, t in m.named_parameters()}
    x64 = x.double().requires_grad_()
    R = heads // kv_heads

    def rot(t):
        return t * cos[:, None].double() + torch.cat((-t[..., D // 2:], t[..., :D // 2]), -1) * sin[:, None].double()

    q = rot((x64 @ P["q_proj.weight"].T).view(B, S, heads, D))
    k = rot((x64 @ P["k_proj.weight"].T).view(B, S, kv_heads, D)).repeat_interleave(R, 2)
    v = (x64 @ P["v_proj.weight"].T).view(B, S, kv_heads, D).repeat_interleave(R, 2)
    at, pad = torch.arange(S), torch.tensor(pads)
    alive = (at[None] >= pad[:, None]).double()
    seen = (at[None] <= at[:, None])[None] & ((at[None, None] >= pad[:, None, None]) | (alive == 0)[:, :, None])
    s = (torch.einsum("bqhd,bkhd->bhqk", q, k) / math.sqrt(D)).masked_fill(~seen[:, None], -math.inf)
    keep = ref.keep_factor(B * heads * S, S, p, 9, 0, 4).view(B, heads, S, S)
    a = torch.einsum("bhqk,bkhd->bqhd", torch.softmax(s, -1) * keep, v) * alive[:, :, None, None]
    want = (a.reshape(B, S, hidden) @ P["o_proj.weight"].T) * ref.keep_factor(B * S, hidden, p, 9, 0, 5).view(B, S, hidden)
    want.backward(cot.double())
    bound = 24 * torch.finfo(ac).eps / 2
    close("y", y.detach(), want.detach(), bound)
    close("dx", xd.grad, x64.grad, bound)
    for n, t in m.named_parameters():
        assert t.grad.dtype == FP32
        close(n, t.grad, P[n].grad, bound)
    # A residual of the block's own type: the sum takes the wider one, as residual + y does.
    with torch.autocast("cuda", ac):
        z, _ = m(xd, (cos.cuda(), sin.cuda()), attention_mask=mask.cuda(), residual=xd)
    assert z.dtype == FP32


@pytest.mark.gpu
@pytest.mark.parametrize("dropout", [0.1, 0.0])
def test_decoder_step_under_autocast_matches_float64(dropout):
    """fp16, u = 2^-11.  Beside the 70 roundings of a model in fp16 (fewer here: stream and norms are fp32), each of
    the 14 products of two blocks rounds its input and its weight, forward and in two gradients: at most 70 + 14 * 6
    = 154 u of a result's norm."""
    pads = [0, 9, 24]
    model = small_model(FP32, dropout, 128, 4, 2).train().fuse_training(seed=77)
    g = torch.Generator().manual_seed(1)
    B, S = 3, 24
    tokens, cot = torch.randn(B, S, 128, generator=g), torch.randn(B, S, 128, generator=g)
    for b, pad in enumerate(pads):
        cot[b, :pad] = 0
    x = tokens.cuda().requires_grad_()
    with torch.autocast("cuda", FP16):
        out, _ = model.model.run_training(x, torch.tensor(pads, dtype=torch.int32, device="cuda"))
    out = out.view(B, S, 128)
    assert out.dtype == FP32
    out.backward(cot.cuda())
    x64, P, want = decoder64(model, tokens, pads, 77, 0)
    want.backward(cot.double())
    bound = 154 * 2.0 ** -11
    alive = (torch.arange(S)[None] >= torch.tensor(pads)[:, None])[..., None]
    close("out", out.detach() * alive.cuda(), want.detach() * alive, bound)
    close("dx", x.grad, x64.grad, bound)
    for name, t in model.model.named_parameters():
        if name.startswith(("layers", "norm", "embed_norm")):
            assert t.grad.dtype == FP32
            close(name, t.grad, P[name].grad, bound)


@pytest.mark.gpu
@pytest.mark.parametrize("ac", [BF16, FP16])
def test_model_step_under_autocast_reaches_every_parameter(ac):
    model = small_model(FP32).train().fuse_training(seed=5)
    data = batch(model, pads=[0, 2, 4])
    targets = data["actions"].masked_fill(data["attention_mask"] == 0, -100)
    with torch.autocast("cuda", ac):
        loss = model(**data, action_targets=targets).loss
    (loss * 1024).backward()  # fp16's gradients, as a loss scaler holds them
    for n, t in model.named_parameters():
        if not n.startswith("value_head"):
            assert t.grad.dtype == FP32 and torch.isfinite(t.grad).all() and (t.grad != 0).any(), n
    # Outside autocast an fp32 model is refused as before.
    with pytest.raises(TypeError, match="training form"):
        model(**data, action_targets=targets)


@pytest.mark.gpu
def test_raw_input_of_a_module_without_a_norm_is_refused():
    from rl_for_mario_b200.attention import FastDTAttention
    from rl_for_mario_b200.dt_model import DTConfig, rope_tables

    cfg = DTConfig(hidden_size=128, num_attention_heads=4, num_key_value_heads=2, context_len=8)
    m = FastDTAttention(cfg).cuda().bfloat16()
    x, pe = torch.zeros(1, 6, 128, device="cuda", dtype=BF16), tuple(t.cuda() for t in rope_tables(32, 6, 1e4))
    for on in (False, True):
        with pytest.raises(ValueError, match="set_fused_norm"):
            m.fuse_training(on)(x, pe, raw_input=True)
    assert m.dropout_state().state_dict()["step"] == 0  # a refused call draws nothing

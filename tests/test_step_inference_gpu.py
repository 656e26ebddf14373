"""A model that is used for inference between training steps computes with the weights that it has.

Every comparison is for equality: the same kernels on the same weights, which are deterministic (cuDNN's convolutions are
told to be)."""
import copy
from types import SimpleNamespace

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def deterministic():
    was = torch.backends.cudnn.deterministic
    torch.backends.cudnn.deterministic = True
    yield
    torch.backends.cudnn.deterministic = was
    from rl_for_mario_b200.kernels import device_status

    torch.cuda.synchronize()
    assert device_status() == 0


def make(qk_norm, state=None):
    from rl_for_mario_b200.dt_model import DTConfig, MarioDT

    torch.manual_seed(0)
    cfg = DTConfig(hidden_size=128, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, context_len=8,
                   dropout=0.0, qk_norm=qk_norm)
    m = MarioDT(cfg).cuda().to(torch.bfloat16).eval()
    if state is not None:
        m.load_state_dict(state)
    return m


def batch(m, B=3, T=5, seed=1):
    g = torch.Generator().manual_seed(seed)
    c = m.config
    d = dict(states=torch.randint(0, 256, (B, T, *c.state_shape), generator=g, dtype=torch.uint8),
             actions=torch.randint(0, c.act_dim, (B, T), generator=g), returns_to_go=torch.rand(B, T, generator=g),
             timesteps=torch.arange(T).expand(B, T))
    return {k: v.cuda() for k, v in d.items()}


def infer(m, b):
    with torch.no_grad():
        return m(**b).action_logits.clone()


@pytest.mark.parametrize("qk_norm", [False, True])
@pytest.mark.parametrize("fused", [False, True])
def test_inference_between_steps(fused, qk_norm):
    m = make(qk_norm).fuse_training()
    if fused:
        m.fuse_norms()
    opt = m.adamw(lr=0.05, weight_decay=0.1, max_norm=1.0)
    b = batch(m)
    seen = [infer(m, b)]
    for _ in range(2):
        m(**b).loss.backward()
        opt.step()
        opt.zero_grad(set_to_none=True)
        seen.append(infer(m, b))
        fresh = make(qk_norm, copy.deepcopy(m.state_dict()))
        if fused:
            fresh.fuse_norms()
        assert torch.equal(seen[-1], infer(fresh, b))
        assert not torch.equal(seen[-1], seen[-2])


def test_a_swapped_module_between_steps():
    from rl_for_mario_b200 import optim
    from rl_for_mario_b200.attention import FastDTAttention
    from rl_for_mario_b200.dt_model import rope_tables

    cfg = SimpleNamespace(hidden_size=128, num_attention_heads=4, num_key_value_heads=2, dropout=0.0, flash_attn=True)
    torch.manual_seed(0)
    m = FastDTAttention(cfg).cuda().bfloat16().fuse_training()
    opt = optim.AdamW(m.parameters(), lr=0.05)
    pe = tuple(t.cuda() for t in rope_tables(32, 16, 1e4))
    x = torch.randn(2, 16, 128, device="cuda").bfloat16()
    with torch.no_grad():
        first = m(x, pe)[0]
    m(x, pe)[0].sum().backward()
    opt.step()
    fresh = FastDTAttention(cfg).cuda().bfloat16()
    fresh.load_state_dict(m.state_dict())
    with torch.no_grad():
        now, want = m(x, pe)[0], fresh(x, pe)[0]
    assert torch.equal(now, want) and not torch.equal(now, first)


def test_inference_after_replays_of_a_captured_step():
    m = make(False).fuse_training().fuse_norms()
    opt = m.adamw(lr=0.05, max_norm=1.0)
    b = batch(m)

    def step():
        m(**b).loss.backward()
        opt.step()
        opt.zero_grad(set_to_none=True)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    infer(m, b)
    for say in (opt.weights_changed, m.weights_changed):
        graph.replay()
        say()
        assert torch.equal(infer(m, b), infer(make(False, copy.deepcopy(m.state_dict())).fuse_norms(), b))
    assert int(opt.steps()) == 3


def test_a_step_between_a_forward_pass_and_its_backward_pass_is_an_error():
    m = make(False).fuse_training()
    opt = m.adamw()
    b = batch(m)
    m(**b).loss.backward()
    loss = m(**b).loss
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_a_captured_inference_after_a_step():
    """The graph reads derived weights where they were at its capture: they are renewed in their place.  A capture that
    finds old ones makes its own at each replay."""
    m = make(True).fuse_training().fuse_norms()
    opt = m.adamw(lr=0.05)
    b = batch(m)
    infer(m, b), infer(m, b)

    def step():
        m(**b).loss.backward()
        opt.step()
        opt.zero_grad(set_to_none=True)

    def captured():
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph), torch.no_grad():
            out = m(**b).action_logits
        return graph, out

    warm = captured()
    step()
    cold = captured()  # the derived weights are those of before the step
    for _ in range(2):
        want = infer(make(True, copy.deepcopy(m.state_dict())).fuse_norms(), b)
        cold[0].replay()
        assert torch.equal(cold[1], want)
        assert torch.equal(infer(m, b), want)
        warm[0].replay()
        assert torch.equal(warm[1], want)
        step()

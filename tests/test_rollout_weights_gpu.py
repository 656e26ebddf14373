"""Rollouts between training steps: graphs and eager steps alike compute with the weights that the model has, with and
without norms of query and key heads."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def deterministic():
    was = torch.backends.cudnn.deterministic
    torch.backends.cudnn.deterministic = True
    yield
    torch.backends.cudnn.deterministic = was


def make(qk_norm, fused, state=None):
    from rl_for_mario_b200.dt_model import DTConfig, MarioDT

    torch.manual_seed(0)
    cfg = DTConfig(hidden_size=128, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, context_len=8,
                   dropout=0.0, qk_norm=qk_norm)
    m = MarioDT(cfg).cuda().to(torch.bfloat16).eval()
    if state is not None:
        m.load_state_dict(state)
    return m.fuse_norms() if fused else m


def inputs(B, T):
    g = torch.Generator().manual_seed(1)
    return (torch.randint(0, 256, (B, T, 4, 84, 84), generator=g, dtype=torch.uint8).cuda(),
            torch.rand(B, T, generator=g).cuda(), torch.arange(T).expand(B, T).cuda())


def episode(ro, states, rtg, ts, actions=None):
    """Logits [T] of an episode in which action t is row t of ``actions``."""
    ro.reset()
    out = []
    for t in range(states.shape[1]):
        a, logits = ro.step(states[:, t], rtg[:, t], ts[:, t])
        if actions is not None:
            ro.prev_action = actions[t]
        out.append(logits.clone())
    return out


@pytest.mark.parametrize("qk_norm", [False, True])
@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("how,episodes", [("adamw", 1), ("torch", 2), ("adamw", 2)])
def test_rollouts_between_steps(how, episodes, fused, qk_norm):
    """Steps from before the graphs are captured on (one episode) or behind that (two); an eager forward pass between
    one of them and the replay.
    The eager rollout of a fresh model with these weights takes its first episode on the same static buffers."""
    from rl_for_mario_b200.rollout import DTRollout

    B, T = 4, 5
    m = make(qk_norm, fused).fuse_training()
    opt = m.adamw(lr=0.02, weight_decay=0.0) if how == "adamw" else torch.optim.AdamW(m.parameters(), lr=0.02)
    states, rtg, ts = inputs(B, T)
    actions = torch.arange(B * T).view(T, B).cuda() % m.config.act_dim
    ro = DTRollout(m, B, T, page_size=16, graphs=True)
    for _ in range(episodes):
        last = episode(ro, states, rtg, ts, actions)
    for turn in range(4):
        m(states, actions.t(), rtg, ts).loss.backward()
        opt.step()
        opt.zero_grad(set_to_none=True)
        if turn == 2:
            with torch.no_grad():
                m(states, actions.t(), rtg, ts)
        got = episode(ro, states, rtg, ts, actions)
        fresh = DTRollout(make(qk_norm, fused, m.state_dict()), B, T, page_size=16, graphs=True)
        want = episode(fresh, states, rtg, ts, actions)
        for t in range(T):
            assert torch.equal(got[t], want[t]), (turn, t, (got[t] - want[t]).abs().max().item())
        assert not torch.equal(got[-1], last[-1])
        last = got
    assert len(ro._graphs) == T


@pytest.mark.parametrize("fused", [False, True])
def test_cached_rollout_with_head_norms_against_prefill(fused):
    """Eager and replayed steps against a forward pass over the whole history.  Logits of bf16 blocks that round at other
    places (two blocks of some ten roundings each, 2^-9 of their size): 40 * 2^-9 of their norm."""
    from rl_for_mario_b200.rollout import DTRollout

    B, T = 4, 6
    m = make(True, fused)
    states, rtg, ts = inputs(B, T)
    actions = torch.arange(B * T).view(T, B).cuda() % m.config.act_dim
    eager = DTRollout(m, B, T, page_size=16)
    graph = DTRollout(m, B, T, page_size=16, graphs=True)
    with torch.no_grad():
        full = m(states, actions.t(), rtg, ts).action_logits.float()
    got = [episode(eager, states, rtg, ts, actions)] + [episode(graph, states, rtg, ts, actions) for _ in range(3)]
    for logits in got:
        for t in range(T):
            off = (logits[t] - full[:, t]).norm() / full[:, t].norm()
            assert off.item() <= 40 * 2.0 ** -9, (t, off.item())
    for a, b in zip(got[1], got[3]):
        assert torch.equal(a, b)

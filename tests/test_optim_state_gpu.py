"""What AdamW.load_state_dict() makes of a rate on the device."""
import copy
import io

import pytest
import torch

pytestmark = pytest.mark.gpu


def one(lr, n=300, seed=0, **kw):
    from rl_for_mario_b200 import optim

    g = torch.Generator().manual_seed(seed)
    p = torch.nn.Parameter(torch.randn(n, generator=g).cuda())
    p.grad = torch.randn(n, generator=g).cuda()
    return p, optim.AdamW([p], lr=lr, weight_decay=0.0, **kw)


def rate(x, shape=()):
    return torch.full(shape, x, device="cuda")


def test_a_loaded_rate_is_the_optimizers_own():
    a, b = one(rate(0.1))[1], one(0.5)[1]
    saved = a.state_dict()
    b.load_state_dict(saved)
    assert isinstance(b.param_groups[0]["lr"], torch.Tensor) and b.param_groups[0]["lr"].item() == pytest.approx(0.1)
    b.param_groups[0]["lr"].fill_(0.7)
    assert a.param_groups[0]["lr"].item() == pytest.approx(0.1)
    assert saved["param_groups"][0]["lr"].item() == pytest.approx(0.1)
    a.param_groups[0]["lr"].fill_(0.2)
    assert b.param_groups[0]["lr"].item() == pytest.approx(0.7)


def test_betas_of_a_loaded_state_are_the_optimizers_own():
    a, b = one(0.1, betas=[0.9, 0.99])[1], one(0.1)[1]
    b.load_state_dict(a.state_dict())
    a.param_groups[0]["betas"][0] = 0.5
    assert list(b.param_groups[0]["betas"]) == [0.9, 0.99]


@pytest.mark.parametrize("bits", [8, 32])
def test_a_checkpoint_on_the_cpu(bits):
    p, a = one(rate(0.1), state_bits=bits)
    a.step()
    f = io.BytesIO()
    torch.save(a.state_dict(), f)
    f.seek(0)
    saved = torch.load(f, map_location="cpu")
    assert not saved["param_groups"][0]["lr"].is_cuda
    q, b = one(rate(0.3, (1,)), state_bits=bits)
    with torch.no_grad():
        q.copy_(p)
    b.load_state_dict(saved)
    a.step(), b.step()
    assert torch.equal(p, q) and int(b.steps()) == 2


@pytest.mark.parametrize("given", ["tensor", "number"])
def test_a_captured_step_reads_the_loaded_rate(given):
    lr = rate(0.25)
    p, a = one(lr)
    a.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    saved = copy.deepcopy(a.state_dict())
    if given == "number":
        saved["param_groups"][0]["lr"] = 0.0625
    else:
        saved["param_groups"][0]["lr"].fill_(0.0625)
    a.load_state_dict(saved)
    assert a.param_groups[0]["lr"] is lr and lr.item() == 0.0625
    q, b = one(0.0625)
    with torch.no_grad():
        q.copy_(p)
    b.load_state_dict({**saved, "param_groups": [{**saved["param_groups"][0], "lr": 0.0625}]})
    graph.replay()
    b.step()
    assert torch.equal(p, q)


def test_a_rate_that_is_refused_changes_nothing():
    p, a = one(0.1)
    a.step()
    saved = copy.deepcopy(a.state_dict())
    for lr in (torch.zeros(2), torch.zeros((), dtype=torch.float64), -1.0):
        saved["param_groups"][0]["lr"] = lr
        saved["state"]["exp_avg"].fill_(7.0)
        with pytest.raises(ValueError, match="lr"):
            a.load_state_dict(saved)
        assert a.param_groups[0]["lr"] == 0.1 and not (a.moments()[0] == 7).any()


def pair(*lr, **kw):
    """An optimizer of two groups with these rates (one: shared)."""
    from rl_for_mario_b200 import optim

    ps = [torch.nn.Parameter(torch.ones(5, device="cuda")) for _ in range(2)]
    if len(lr) == 1:
        return optim.AdamW([dict(params=[p]) for p in ps], lr=lr[0])
    return optim.AdamW([dict(params=[p], lr=x) for p, x in zip(ps, lr)])


@pytest.mark.parametrize("where", ["cuda", "cpu"])
def test_groups_that_share_a_rate(where):
    def rates(o):
        return [round(float(g["lr"]), 4) for g in o.param_groups]

    def saved(o):
        s = o.state_dict()
        if where == "cpu":
            f = io.BytesIO()
            torch.save(s, f)
            f.seek(0)
            s = torch.load(f, map_location="cpu")
        return s

    shared, apart = saved(pair(rate(0.125))), saved(pair(rate(0.25), rate(0.5)))
    for make in (lambda: pair(0.75), lambda: pair(rate(0.75))):
        o = make()
        o.load_state_dict(shared)
        assert rates(o) == [0.125, 0.125]
        o.param_groups[0]["lr"].fill_(0.0625)  # one rate still
        assert rates(o) == [0.0625, 0.0625]
        o = make()
        o.load_state_dict(apart)
        assert rates(o) == [0.25, 0.5]
        o.param_groups[0]["lr"].fill_(1.0)
        assert rates(o) == [1.0, 0.5]
    o = pair(rate(0.75), rate(1.0))
    own = [g["lr"] for g in o.param_groups]
    o.load_state_dict(shared)
    assert rates(o) == [0.125, 0.125] and all(g["lr"] is t for g, t in zip(o.param_groups, own))

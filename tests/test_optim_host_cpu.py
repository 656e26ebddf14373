"""The optimizer's host side on CPU tensors: its launch is replaced by writes through the addresses that the entry
point gets, as the kernel's are.  (AdamW refuses CPU parameters; the check is taken out here.)"""
import copy
import ctypes
import pickle

import pytest
import torch

from rl_for_mario_b200 import kernels, optim


class Calls(list):
    """The arguments of the launches: a dict of each."""

    def __call__(self, name, dev, count, at, to, sizes, kinds, ngroups, groups, bits, *rest):
        assert name == "dt_adamw_step"

        def longs(p):
            return list((ctypes.c_int64 * count).from_address(p))

        call = dict(count=count, at=longs(at), to=longs(to), sizes=longs(sizes), ngroups=ngroups,
                    groups=[optim._GROUP.unpack_from(groups, i * optim._GROUP.size) for i in range(ngroups)])
        for p, g, n in zip(call["at"], call["to"], call["sizes"]):
            if g:  # fp32 weights: p -= g
                for i in range(n):
                    w = ctypes.c_float.from_address(p + 4 * i)
                    w.value -= ctypes.c_float.from_address(g + 4 * i).value
        self.append(call)


@pytest.fixture
def calls(monkeypatch):
    c = Calls()
    monkeypatch.setattr(optim.AdamW, "_check_param", lambda self, p: None)
    monkeypatch.setattr(kernels, "_launch", c)
    return c


def params(*shapes):
    return [torch.nn.Parameter(torch.ones(s)) for s in shapes]


def test_a_step_raises_the_versions_of_what_it_wrote(calls):
    ps = params(3, (2, 5), 4)
    opt = optim.AdamW(ps)
    ps[0].grad, ps[2].grad = torch.full((3,), 0.5), torch.full((4,), 0.25)
    was = [p._version for p in ps]
    opt.step()
    assert len(calls) == 1 and (ps[0] == 0.5).all() and (ps[1] == 1).all() and (ps[2] == 0.75).all()
    now = [p._version for p in ps]
    assert now[0] > was[0] and now[1] == was[1] and now[2] > was[2]
    for p in ps:
        p.grad = None
    opt.step()  # no gradient: no step
    assert len(calls) == 1 and [p._version for p in ps] == now
    opt.weights_changed()
    assert all(p._version > v for p, v in zip(ps, now))


def test_a_step_between_a_forward_pass_and_its_backward_pass_is_an_error(calls):
    ps = params((4, 3))
    opt = optim.AdamW(ps)
    ps[0].grad = torch.ones(4, 3)
    x = torch.ones(2, 3, requires_grad=True)
    y = torch.nn.functional.linear(x, ps[0]).sum()
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@pytest.mark.parametrize("make", [list, tuple])
def test_every_step_takes_the_groups_numbers_as_they_are(calls, make):
    ps = params(3, 4)
    ps[0].grad, ps[1].grad = torch.ones(3), torch.ones(4)
    opt = optim.AdamW([dict(params=[ps[0]], betas=make((0.9, 0.99))), dict(params=[ps[1]])], betas=make((0.8, 0.98)))
    opt.step()
    group = opt.param_groups[0]
    if make is list:
        group["betas"][0] = 0.5
    else:
        group["betas"] = (0.5, 0.99)
    opt.step()
    group["lr"], group["eps"], group["weight_decay"] = 0.25, 1e-3, 0.125
    opt.step()
    first = [c["groups"][0][:5] for c in calls]
    assert first == [(1e-3, 0.9, 0.99, 1e-8, 1e-2), (1e-3, 0.5, 0.99, 1e-8, 1e-2), (0.25, 0.5, 0.99, 1e-3, 0.125)]
    assert all(c["groups"][1][:5] == (1e-3, 0.8, 0.98, 1e-8, 1e-2) for c in calls)
    group["betas"] = make((1.0, 0.99))
    with pytest.raises(ValueError, match="betas"):
        opt.step()
    assert len(calls) == 3


def test_a_group_without_parameters_added_later(calls):
    ps = params(3, 4)
    ps[0].grad, ps[1].grad = torch.ones(3), torch.ones(4)
    opt = optim.AdamW([ps[0]])
    opt.step()
    opt.add_param_group(dict(params=[], lr=0.5))
    opt.step()
    assert [c["ngroups"] for c in calls] == [1, 2] and calls[1]["groups"][1][0] == 0.5
    opt.add_param_group(dict(params=[ps[1]], lr=0.25))
    opt.step()
    assert calls[2]["ngroups"] == 3 and calls[2]["sizes"] == [3, 4] and calls[2]["groups"][2][0] == 0.25
    assert [len(g["params"]) for g in opt.state_dict()["param_groups"]] == [1, 0, 1]


@pytest.mark.parametrize("how", ["all gradients", "one missing", "another order of memory"])
def test_moved_parameters_that_share_memory_are_refused(calls, how):
    ps = params(6, 5, 4)
    if how == "another order of memory":
        ps.append(torch.nn.Parameter(torch.ones(2, 3, 4, 5).to(memory_format=torch.channels_last)))
    opt = optim.AdamW(ps)
    for p in ps:
        p.grad = torch.ones_like(p)
    opt.step()
    if how == "one missing":
        ps[2].grad = None
    pool = torch.zeros(64)
    for p, at in zip(ps, (0, 5, 32)):  # the last element of the first is the first of the second
        p.data = pool[at:at + p.numel()]
    with pytest.raises(ValueError, match="share memory"):
        opt.step()
    assert len(calls) == 1
    for p, at in zip(ps, (0, 6, 32)):
        p.data = pool[at:at + p.numel()]
    opt.step()
    assert len(calls) == 2 and calls[1]["at"][:3] == [pool.data_ptr() + 4 * n for n in (0, 6, 32)]
    ps[1].data = torch.zeros(7)
    with pytest.raises(ValueError, match="changed"):
        opt.step()


def test_memory_that_a_parameter_left_is_given_back(calls):
    import weakref

    ps = params(6, 5)
    opt = optim.AdamW(ps)
    for p in ps:
        p.grad = torch.ones_like(p)
    opt.step()
    old = weakref.ref(ps[0].data.untyped_storage())
    assert old() is not None
    ps[0].data = torch.zeros(6)  # as a model that is moved elsewhere
    assert old() is None


@pytest.mark.parametrize("how", ["smaller", "larger type"])
def test_a_parameter_of_another_size_at_its_old_address_is_refused(calls, how, monkeypatch):
    """What was there may have been given back and handed out anew: an address alone says nothing."""
    pool = torch.ones(64)
    p = torch.nn.Parameter(pool[:8] if how == "smaller" else pool[:8].view(torch.bfloat16)[:8])
    opt = optim.AdamW([p])
    p.grad = torch.ones_like(p)
    monkeypatch.setattr(optim, "_on", lambda t: None)  # (a CPU tensor's index is not None)
    opt._ready()
    opt._addresses(opt._order, None)
    g = p.grad
    p.grad = None
    p.data = pool[:4] if how == "smaller" else pool[:8]
    monkeypatch.setattr(optim, "_grad_of", lambda t: g)
    assert p.data_ptr() == pool.data_ptr()
    with pytest.raises(ValueError, match="changed"):
        opt._addresses(opt._order, None)


def test_hooks_of_saving_and_loading_are_called(calls):
    ps = params(3)
    opt = optim.AdamW(ps, lr=0.5)
    seen = []
    handles = [opt.register_state_dict_pre_hook(lambda o: seen.append(("save", o))),
               opt.register_state_dict_post_hook(lambda o, s: {**s, "more": 7}),
               opt.register_load_state_dict_pre_hook(lambda o, s: {k: v for k, v in s.items() if k != "more"}),
               opt.register_load_state_dict_pre_hook(lambda o, s: s["param_groups"][0].update(lr=0.125)),
               opt.register_load_state_dict_post_hook(lambda o: seen.append(("load", o)))]
    saved = opt.state_dict()
    assert saved["more"] == 7 and seen == [("save", opt)]
    opt.load_state_dict(saved)
    assert opt.param_groups[0]["lr"] == 0.125 and seen == [("save", opt), ("load", opt)] and saved["more"] == 7
    for h in handles:
        h.remove()
    assert "more" not in opt.state_dict() and len(seen) == 2


@pytest.mark.parametrize("how", ["deepcopy", "pickle"])
def test_a_copy_is_an_optimizer_of_its_own(calls, how):
    """With a scheduler, which replaces step() of the object, and hooks that cannot be pickled."""
    ps = params(6, 5)
    opt = optim.AdamW([dict(params=[ps[0]], betas=[0.9, 0.99]), dict(params=[ps[1]])], lr=0.5)
    torch.optim.lr_scheduler.LambdaLR(opt, lambda t: 1.0)
    seen = []
    opt.register_step_post_hook(lambda *x: seen.append("step"))
    opt.register_state_dict_pre_hook(lambda *x: seen.append("save"))
    for p in ps:
        p.grad = torch.ones_like(p)
    opt.step()
    other = copy.deepcopy(opt) if how == "deepcopy" else pickle.loads(pickle.dumps(opt))
    qs = [p for g in other.param_groups for p in g["params"]]
    assert seen == ["step"] and len(calls) == 1
    for q in qs:
        assert all(q is not p for p in ps)
        q.grad = torch.full_like(q, 0.5)
    other.param_groups[0]["betas"][0] = 0.75
    other.step()
    assert seen == ["step"] and len(calls) == 2
    assert calls[1]["at"] == [q.data_ptr() for q in qs] and calls[1]["groups"][0][1] == 0.75
    assert all((p == 0).all() for p in ps) and all((q == -0.5).all() for q in qs)
    other.state_dict()
    opt.step()
    assert seen == ["step", "step"] and calls[2]["at"] == [p.data_ptr() for p in ps]
    assert calls[2]["groups"][0][1] == 0.9
    with torch.no_grad():
        other.moments()[0].fill_(3.0)
    assert not (opt.moments()[0] == 3).any()

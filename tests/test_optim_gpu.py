"""AdamW and the gradient's norm over many tensors against their restatement (oracle/step_ref.py).

Tolerances, elementwise.  With e = 2^-24: m' is two products of rounded factors and a sum, of a gradient
that clipping (norm 2 e, its sum, division and product) may have moved by 6 e: 12 e on the absolute terms.
v' the same with the gradient squared: 20 e on v' (all its terms are positive).  A step is rate m' / (root
sqrt(v') + eps): 12 e of m', 10 e of the root of v', 2 + 2 e of sqrt and its factor, 2 e of the sum, 4 e of the
division, 3 e of the rate and its product: 40 e on the step's absolute terms; a weight takes two products
and a sum, 4 e, and its own rounding where it has 16 bits.  In 8 bits the codes are whole numbers and equal
the restatement's, whose averages are float32 with the kernel's roundings.
"""
import copy
import math

import numpy as np
import pytest
import torch

from oracle import step_ref as ref

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
E = 2.0 ** -24
pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_device_error():
    yield
    from rl_for_mario_b200.kernels import device_status

    torch.cuda.synchronize()
    assert device_status() == 0


def near(name, got, want, tol):
    got = got.detach().double().cpu()
    assert torch.isfinite(got).all(), name
    over = ((got - want).abs() - tol).max().item() if got.numel() else 0.0
    assert over <= 0, f"{name}: {over:.3e} over its bound"


# ------------------------------------------------------------------------------------------- norm
NORMS = [([1], [FP32]), ([0, 3, 0], [BF16]), ([255, 256, 257, 1023, 1024, 1025], [BF16, FP32, FP16]),
         ([1 << 20, 7, 300001], [FP32, BF16]), ([5] * 959 + [4097] * 3, [FP16, FP32]), ([3] * 2000, [BF16]),
         ([0] * 800 + [5], [FP32]), ([7] + [0] * 1600, [BF16])]


@pytest.mark.parametrize("sizes,types", NORMS)
def test_norm(sizes, types):
    from rl_for_mario_b200 import optim

    g = torch.Generator().manual_seed(1)
    ts = [torch.randn(n, generator=g).to(types[i % len(types)]) for i, n in enumerate(sizes)]
    want = math.sqrt(sum(t.double().pow(2).sum().item() for t in ts))
    got = optim.grad_norm([t.cuda() for t in ts])
    assert got.dtype == FP32 and got.dim() == 0
    # Two squares and their sum in fp32, 3 e on positive terms, halved by the root; fp64 behind them; one rounding.
    assert abs(got.item() - want) <= want * 5 * E


def test_norm_of_any_layout_and_size_of_number():
    from rl_for_mario_b200 import optim

    x = torch.randn(40, 30, 20, device="cuda")
    views = [x, x.permute(2, 0, 1), x[:, ::2], x[3:, 5:, 7:], x[:1].expand(7, 30, 20), None,
             torch.randn(10001, device="cuda").bfloat16()[1:]]
    want = math.sqrt(sum(t.double().pow(2).sum().item() for t in views if t is not None))
    assert abs(optim.grad_norm(views).item() - want) <= want * 5 * E
    for size in (1e30, 1e18, 1e-19, 1e-25, 1e-38):
        y = torch.randn(5000, device="cuda").mul_(size)
        want = y.double().pow(2).sum().sqrt().item()
        got = optim.grad_norm([y, torch.zeros(3000, device="cuda")]).item()
        assert abs(got - want) <= want * 5 * E + 2.0 ** -149, size
    assert optim.grad_norm([torch.zeros(0, device="cuda")]).item() == 0
    assert math.isnan(optim.grad_norm([x, torch.tensor([math.nan], device="cuda")]).item())
    assert optim.grad_norm([x, torch.tensor([-math.inf], device="cuda").half()]).item() == math.inf
    with pytest.raises(ValueError, match="one tensor"):
        optim.grad_norm([None])
    with pytest.raises(ValueError, match="CUDA|devices"):
        optim.grad_norm([x, torch.zeros(3)])
    with pytest.raises(TypeError, match="dtype"):
        optim.grad_norm([x.double()])


# ------------------------------------------------------------------------------------------- step
def blocks_of(params):
    at = [0]
    for p in params:
        at.append(at[-1] + (p.numel() + 255) // 256 * 256)
    return at


def part(flat, at, p):
    """A parameter's piece of a flat array, in the parameter's order of memory."""
    return flat[at:at + p.numel()]


def memory(t):
    return torch.as_strided(t.detach(), (t.numel(),), (1,))


SHAPES = [(1,), (256,), (257,), (3, 5, 7), (64, 32), (1000, 33), (0,), (2049,), (31, 33, 3)]
RUNS = [
    # dtypes, bits, master, max_norm, lr, betas, eps, wd
    ([FP32], 32, False, None, 1e-3, (0.9, 0.999), 1e-8, 0.1),
    ([BF16], 32, False, 0.5, 1e-2, (0.8, 0.95), 1e-6, 0.0),
    ([FP16, BF16, FP32], 32, True, 1e9, 3e-4, (0.9, 0.98), 1e-8, 0.3),
    ([FP16], 32, False, None, 1e-3, (0.0, 0.0), 1e-3, 0.01),
    ([FP32], 8, False, None, 1e-3, (0.9, 0.999), 1e-8, 0.1),
    ([BF16, FP32, FP16], 8, True, 0.25, 1e-2, (0.95, 0.99), 1e-8, 0.2),
    ([BF16], 8, False, 1e6, 1e-2, (0.9, 0.999), 1e-8, 0.0),
]


def make_params(dtypes, seed=0):
    g = torch.Generator().manual_seed(seed)
    ps = [torch.nn.Parameter((torch.randn(s, generator=g) * 0.05).to(dtypes[i % len(dtypes)]).cuda())
          for i, s in enumerate(SHAPES)]
    # Order of memory other than that of the dimensions.
    conv = torch.randn(8, 3, 5, 5, generator=g).to(dtypes[0]).cuda().to(memory_format=torch.channels_last)
    return ps + [torch.nn.Parameter(conv)]


def set_grads(ps, seed):
    g = torch.Generator().manual_seed(seed)
    for i, p in enumerate(ps):
        # Sizes from 1e-6 to 1, some zeros; a few parameters have no gradient now and then.
        x = torch.randn(p.shape, generator=g) * torch.exp(torch.randn(p.shape, generator=g) * 2 - 5)
        x = torch.where(torch.rand(p.shape, generator=g) < 0.1, torch.zeros(()), x).to(p.dtype).cuda()
        p.grad = None if (i + seed) % 7 == 6 else x.to(memory_format=torch.channels_last) if x.dim() == 4 else x


def adamw(ps, groups=None, **kw):
    from rl_for_mario_b200 import optim

    return optim.AdamW(groups or ps, **kw)


@pytest.mark.parametrize("dtypes,bits,master,max_norm,lr,betas,eps,wd", RUNS)
def test_steps(dtypes, bits, master, max_norm, lr, betas, eps, wd):
    ps = make_params(dtypes)
    cut = 4
    groups = [dict(params=ps[:cut]), dict(params=ps[cut:], weight_decay=wd / 2, lr=lr * 2, betas=(betas[0] / 2, betas[1]))]
    opt = adamw(ps, groups, lr=lr, betas=betas, eps=eps, weight_decay=wd, state_bits=bits, master=master,
                max_norm=max_norm, seed=99)
    at = blocks_of(ps)
    for t in (1, 2, 3):
        set_grads(ps, t)
        before = copy.deepcopy(opt.state_dict()["state"])
        old = [memory(p).cpu() for p in ps]
        grads = [None if p.grad is None else memory(p.grad).cpu() for p in ps]
        old_m, old_v = (x.float().cpu() for x in opt.moments())
        opt.step()
        m, v = opt.moments()
        after = opt.state_dict()["state"]
        assert int(opt.steps()) == t == int(after["step"])
        clip = 1.0
        if max_norm is not None:
            norm = math.sqrt(sum(x.double().pow(2).sum().item() for x in grads if x is not None))
            assert abs(opt.norm.item() - norm) <= norm * 5 * E
            clip = min(1.0, max_norm / (norm + 1e-6))
            clip32 = np.minimum(np.float32(1), np.float32(max_norm) / (np.float32(opt.norm.item()) + np.float32(1e-6)))
        if bits == 8:
            words = ref.step_words(at[-1], 99, t)
        for i, p in enumerate(ps):
            sl = slice(at[i], at[i] + (p.numel() + 255) // 256 * 256)
            if grads[i] is None:
                assert torch.equal(memory(p).cpu(), old[i])
                for k in before:
                    if k.startswith("exp") or k == "master":
                        s2 = slice(sl.start // 256, sl.stop // 256) if k.endswith("scale") else sl
                        assert torch.equal(before[k][s2], after[k][s2])
                continue
            b1, b2 = betas if i < cut else (betas[0] / 2, betas[1])
            rate, decay = (lr, wd) if i < cut else (lr * 2, wd / 2)
            kept = master and p.dtype != FP32
            w = part(before["master"], at[i], p).cpu() if kept else old[i]
            r = ref.adamw(w, grads[i], part(old_m, at[i], p), part(old_v, at[i], p), t, rate, b1, b2, eps, decay, clip)
            (want, (ap, au)) = r["p"]
            tol = 4 * E * ap + 40 * E * au + E * want.abs()
            if kept:
                near("master", part(after["master"], at[i], p), want, tol)
                assert torch.equal(memory(p), part(after["master"], at[i], p).to(p.dtype))
            else:
                u = 0 if p.dtype == FP32 else torch.finfo(p.dtype).eps / 2
                tiny = 2.0 ** -25 if p.dtype == FP16 else 0.0
                near("p", memory(p), want, tol * (1 + u) + u * want.abs() + tiny)
            if bits == 32:
                near("m", part(m, at[i], p), r["m"][0], 12 * E * r["m"][1] + 2.0 ** -149)
                near("v", part(v, at[i], p), r["v"][0], 20 * E * r["v"][1] + 2.0 ** -149)
                continue
            pad = sl.stop - sl.start - p.numel()
            g = np.pad(grads[i].float().numpy(), (0, pad))
            m1, v1 = ref.averages_f32(old_m[sl].numpy(), old_v[sl].numpy(), g, b1, b2,
                                      None if max_norm is None else clip32)
            for name, x, word, kind in (("exp_avg", m1, words[0], ref.FIRST), ("exp_avg_sq", v1, words[1], ref.SECOND)):
                codes, scales = ref.encode(x, word[sl], kind)
                got = after[name][sl].cpu().numpy()
                assert np.array_equal(after[name + "_scale"][sl.start // 256:sl.stop // 256].cpu().numpy(), scales)
                assert np.array_equal(got, codes), (name, i, int((got != codes).sum()))
                value = (m if name == "exp_avg" else v)[sl].float().cpu().numpy()
                assert np.array_equal(value, ref.decode(codes, scales, kind))


@pytest.mark.parametrize("dtype,master", [(BF16, False), (FP16, True), (FP32, False)])
def test_large_units_of_8_bit_averages(dtype, master):
    """Enough elements for units of eight blocks: whole ones, ones that a tensor ends in, tensors of less than one, an
    address off the boundary.  Codes, scales and weights of windows of each against the restatement."""
    sizes = [24_000_003, 5, 256 * 9, 700_001, 2048, 1]
    g = torch.Generator(device="cuda").manual_seed(0)
    pool = torch.randn(sum(sizes) + 64, generator=g, device="cuda").mul_(0.05).to(dtype)
    ps, at = [], 0
    for i, n in enumerate(sizes):
        at += 1 if i == 3 else (-at) % 8
        ps.append(torch.nn.Parameter(pool[at:at + n]))
        at += n
    opt = adamw(ps, lr=1e-2, state_bits=8, master=master, weight_decay=0.1, seed=7)
    starts = blocks_of(ps)
    for t in (1, 2):
        for p in ps:
            p.grad = torch.randn(p.shape, generator=g, device="cuda").mul_(1e-3).to(dtype)
        old = [p.detach().cpu() for p in ps]
        state = {k: v.cpu().clone() for k, v in opt.state_dict()["state"].items() if isinstance(v, torch.Tensor)}
        opt.step()
        after = {k: v.cpu() for k, v in opt.state_dict()["state"].items() if isinstance(v, torch.Tensor)}
        for i, (p, n) in enumerate(zip(ps, sizes)):
            blocks = (n + 255) // 256
            for b0 in sorted({0, max(0, blocks // 2 - 8), max(0, blocks - 24)}):
                b1 = min(blocks, b0 + 24)
                lo, hi = b0 * 256, min(n, b1 * 256)
                first = starts[i] // 256 + b0
                sl, sb = slice(first * 256, (first + b1 - b0) * 256), slice(first, first + b1 - b0)
                m0 = ref.decode(state["exp_avg"][sl].numpy(), state["exp_avg_scale"][sb].numpy(), ref.FIRST)
                v0 = ref.decode(state["exp_avg_sq"][sl].numpy(), state["exp_avg_sq_scale"][sb].numpy(), ref.SECOND)
                x = p.grad[lo:hi].cpu()
                m1, v1 = ref.averages_f32(m0, v0, np.pad(x.float().numpy(), (0, len(m0) - len(x))), 0.9, 0.999)
                block = np.arange(first * 32, (first + b1 - b0) * 32, dtype=np.uint64)
                w = ref.philox_words(block, 7, t, ref.SITE).reshape(-1).astype(np.int64)
                for name, y, words, kind in (("exp_avg", m1, (w >> 8) | ((w & 255) << 8), ref.FIRST), ("exp_avg_sq", v1, w, ref.SECOND)):
                    codes, scales = ref.encode(y, words, kind)
                    assert np.array_equal(after[name][sl].numpy(), codes) and np.array_equal(after[name + "_scale"][sb].numpy(), scales)
                kept = master and dtype != FP32
                r = ref.adamw(state["master"][sl][:hi - lo] if kept else old[i][lo:hi], x, torch.from_numpy(m0[:hi - lo]),
                              torch.from_numpy(v0[:hi - lo]), t, 1e-2, 0.9, 0.999, 1e-8, 0.1)
                want, (ap, au) = r["p"]
                tol, u = 4 * E * ap + 40 * E * au + E * want.abs(), 0 if kept or dtype == FP32 else torch.finfo(dtype).eps / 2
                near("p", after["master"][sl][:hi - lo] if kept else p[lo:hi], want, tol * (1 + u) + u * want.abs())
                if kept:
                    assert torch.equal(p[lo:hi].cpu(), after["master"][sl][:hi - lo].to(dtype))
    assert int(opt.steps()) == 2


def test_a_step_that_is_not_finite_changes_nothing():
    for bits in (8, 32):
        ps = make_params([BF16])
        opt = adamw(ps, state_bits=bits, master=True, max_norm=1.0)
        set_grads(ps, 1)
        opt.step()
        for bad in (math.nan, math.inf):
            set_grads(ps, 2)
            ps[5].grad[3, 3] = bad
            was, old = copy.deepcopy(opt.state_dict()["state"]), [p.detach().clone() for p in ps]
            opt.step()
            assert not math.isfinite(opt.norm.item()) and int(opt.steps()) == 1
            now = opt.state_dict()["state"]
            assert all(torch.equal(was[k], now[k]) for k in was if k != "seed")
            assert all(torch.equal(a, b) for a, b in zip(old, ps))
        set_grads(ps, 3)
        opt.step()
        assert int(opt.steps()) == 2
    # Without clipping nothing is looked at: NaN in its element, in 8 bits from the next step on in its block.
    p = torch.nn.Parameter(torch.ones(600, device="cuda"))
    for bits in (32, 8):
        with torch.no_grad():
            p.fill_(1.0)
        opt = adamw([p], state_bits=bits)
        p.grad = torch.ones(600, device="cuda")
        p.grad[300] = math.nan
        opt.step()
        assert torch.isnan(p).nonzero().flatten().tolist() == [300]
        p.grad = torch.ones(600, device="cuda")
        opt.step()
        bad = torch.isnan(p).nonzero().flatten().tolist()
        assert bad == ([300] if bits == 32 else list(range(256, 512)))


def test_many_tensors_and_layouts():
    """More tensors than a launch takes; addresses off every boundary; gradients in another order of memory."""
    g = torch.Generator().manual_seed(5)
    pool = torch.randn(60000, generator=g).cuda()
    ps, gs, at = [], [], 1
    for i in range(2100):
        n = 1 + i % 11
        ps.append(torch.nn.Parameter(pool[at:at + n]))
        gs.append(torch.randn(n, generator=g).cuda())
        at += n + i % 3
    ps.append(torch.nn.Parameter(pool[at:at + 35 * 20].view(35, 20).t()))
    gs.append(torch.randn(20, 35, generator=g).cuda())
    for p, x in zip(ps, gs):
        p.grad = x
    old = pool.cpu()
    opt = adamw(ps, lr=0.01, weight_decay=0.5, max_norm=3.0)
    opt.step()
    norm = math.sqrt(sum(x.double().pow(2).sum().item() for x in gs))
    assert abs(opt.norm.item() - norm) <= norm * 5 * E
    new = pool.cpu()
    touched = torch.zeros(60000, dtype=torch.bool)
    for p, x in zip(ps, gs):
        o = p.storage_offset()
        touched[o:o + p.numel()] = True
        w = torch.as_strided(old, p.shape, p.stride(), o)
        r = ref.adamw(w, x.cpu(), torch.zeros(p.shape), torch.zeros(p.shape), 1, 0.01, 0.9, 0.999, 1e-8, 0.5, 3.0 / (norm + 1e-6))
        want, (ap, au) = r["p"]
        near("p", p, want, 4 * E * ap + 40 * E * au + E * want.abs())
    assert torch.equal(old[~touched], new[~touched]) and touched.any()
    assert int(opt.steps()) == 1


def test_group_added_later_and_state_across_optimizers():
    for bits in (8, 32):
        ps = make_params([BF16, FP32])
        one = adamw(ps[:4], state_bits=bits, master=True, seed=-3, lr=0.01)
        set_grads(ps, 1)
        one.step()
        kept = copy.deepcopy(one.state_dict()["state"])
        one.add_param_group(dict(params=ps[4:], lr=0.02))
        now = one.state_dict()["state"]
        for k, t in kept.items():
            if k not in ("seed", "step"):
                assert torch.equal(now[k][:t.numel()], t)
        set_grads(ps, 2)
        # The same step from a loaded state, on copies of the parameters.
        qs = [torch.nn.Parameter(p.detach().clone(memory_format=torch.preserve_format)) for p in ps]
        for p, q in zip(ps, qs):
            q.grad = None if p.grad is None else p.grad.clone(memory_format=torch.preserve_format)
        two = adamw(qs, [dict(params=qs[:4]), dict(params=qs[4:])], state_bits=bits, master=True)
        two.load_state_dict(copy.deepcopy(one.state_dict()))
        assert two.param_groups[1]["lr"] == 0.02 and two.param_groups[0]["params"][0] is qs[0]
        one.step(), two.step()
        for p, q in zip(ps, qs):
            assert torch.equal(p, q)
        a, b = one.state_dict()["state"], two.state_dict()["state"]
        assert all(torch.equal(torch.as_tensor(a[k]), torch.as_tensor(b[k])) for k in a)
        wrong = adamw(qs[:3], state_bits=bits, master=True)
        with pytest.raises(ValueError, match="groups"):
            wrong.load_state_dict(one.state_dict())
        with pytest.raises(ValueError, match="state has"):
            adamw(qs, [dict(params=qs[:4]), dict(params=qs[4:])], state_bits=40 - bits).load_state_dict(one.state_dict())


def test_fp32_weights_taken_anew():
    ps = make_params([BF16, FP32])
    opt = adamw(ps, master=True, lr=0.0, weight_decay=0.0)
    set_grads(ps, 1)
    opt.step()
    with torch.no_grad():
        for p in ps:
            p.mul_(3.0)
    now = [p.detach().clone() for p in ps]
    opt.reset_master()
    set_grads(ps, 2)
    opt.step()  # a rate of zero: the weights are what they were set to
    for p, q in zip(ps, now):
        assert torch.equal(p, q)
    at = blocks_of(ps)
    for i, p in enumerate(ps):
        want = torch.zeros(p.numel(), device="cuda") if p.dtype == FP32 else memory(p).float()
        assert torch.equal(part(opt.master, at[i], p), want)
    for p in ps:
        p.grad = None
    opt.step()
    assert int(opt.steps()) == 2


def test_captured_step_reads_rate_number_and_gradient_anew():
    for bits in (32, 8):
        lr = torch.full((), 0.01, device="cuda")
        ps, qs = make_params([BF16]), make_params([BF16])
        a = adamw(ps, lr=lr, state_bits=bits, max_norm=1.0, seed=4)
        b = adamw(qs, lr=0.01, state_bits=bits, max_norm=1.0, seed=4)
        held = []
        for p in ps:
            p.grad = torch.zeros_like(p)
            held.append(p.grad)
        a.state_dict()  # the flat arrays are made before the capture
        a.step()        # gradients of zero: averages stay zero; decay alone
        for q in qs:
            q.grad = torch.zeros_like(q)
        b.step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            a.step()
        for t in range(1, 4):
            set_grads(qs, 7 * t + 1)  # (a parameter without a gradient has one of zeros in neither: see below)
            for q, h in zip(qs, held):
                if q.grad is None:
                    q.grad = torch.zeros_like(q)
                h.copy_(q.grad)
            b.param_groups[0]["lr"] = float(np.float32(0.01 / t))
            lr.fill_(b.param_groups[0]["lr"])
            graph.replay()
            b.step()
            assert int(a.steps()) == t + 1 == int(b.steps())
            for p, q in zip(ps, qs):
                assert torch.equal(p, q)
            assert all(torch.equal(x, y) for x, y in zip(a.moments(), b.moments()))


def test_hooks_closure_and_scheduler():
    ps, qs = make_params([FP32]), make_params([FP32])
    a, b = adamw(ps, lr=0.1), adamw(qs, lr=0.1)
    seen = []
    handles = [a.register_step_pre_hook(lambda *x: seen.append("pre")), a.register_step_post_hook(lambda *x: seen.append("post"))]
    half = torch.optim.lr_scheduler.LambdaLR(a, lambda t: 0.5 ** t)

    def closure():
        seen.append(torch.is_grad_enabled())
        set_grads(ps, 1)
        return 7.0

    assert a.step(closure) == 7.0 and seen == ["pre", True, "post"]
    half.step()
    assert a.param_groups[0]["lr"] == 0.05
    for h in handles:
        h.remove()
    set_grads(ps, 2)
    assert a.step() is None and len(seen) == 3
    set_grads(qs, 1)
    b.step()
    b.param_groups[0]["lr"] = 0.05
    set_grads(qs, 2)
    b.step()
    for p, q in zip(ps, qs):
        assert torch.equal(p, q)
    c = copy.deepcopy(a)
    assert c.param_groups[0]["params"][0] is not ps[0] and int(c.steps()) == 2
    with torch.no_grad():
        ps[0].add_(1.0)
    assert not torch.equal(c.param_groups[0]["params"][0], ps[0])


def test_another_stream():
    ps, qs = make_params([FP32]), make_params([FP32])
    a, b = adamw(ps, max_norm=1.0), adamw(qs, max_norm=1.0)
    set_grads(ps, 1), set_grads(qs, 1)
    a.step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b.step()
    side.synchronize()
    for p, q in zip(ps, qs):
        assert torch.equal(p, q)


def test_averages_in_8_bits_follow_those_in_32():
    """Gradients of one size for 3,000 steps.  Unbiased rounding: over 65,536 elements the mean of v8 / v32 is 1 up to
    its spread / 256.  Spread: a step moves v by d = 0.001 |x - 1| v, x = g^2 / v, to which rounding at random to a
    spacing of up to 1/8 v adds a variance of up to d v / 8; over the memory of 1,000 steps, half of it counting,
    500 * 0.001 * E|x - 1| / 8 = 0.06 at most (E|x - 1| = 0.97): 0.25 of v."""
    from rl_for_mario_b200 import optim

    n = 65536
    p8, p32 = (torch.nn.Parameter(torch.zeros(n, device="cuda")) for _ in range(2))
    o8 = optim.AdamW([p8], lr=0.0, state_bits=8, seed=1)
    o32 = optim.AdamW([p32], lr=0.0)
    g = torch.Generator(device="cuda").manual_seed(0)
    for _ in range(3000):
        p8.grad = p32.grad = torch.randn(n, generator=g, device="cuda").mul_(1e-3)
        o8.step(), o32.step()
    (m8, v8), (m32, v32) = ([x.float() for x in o.moments()] for o in (o8, o32))
    ratio = v8 / v32
    spread = ratio.std().item()
    assert spread <= 0.25 and abs(ratio.mean().item() - 1) <= 5 * 0.25 / 256
    # m: each step rounds anew, variance up to (|m| / 8)^2 / 4; 1 / (1 - 0.81) of them are remembered.  Near a block's
    # zero steps are those of its subnormal numbers, 2^-16 of its largest value.
    off = (m8 - m32).pow(2).mean().sqrt() / m32.pow(2).mean().sqrt()
    assert off.item() <= 0.0625 / math.sqrt(0.19) and abs((m8 - m32).mean().item()) <= 5 * 1e-3 * 0.25 / 256


def test_refusals():
    from rl_for_mario_b200 import optim

    p = torch.nn.Parameter(torch.zeros(10, 10, device="cuda"))
    ok = dict(params=[p])
    for kw, match in ((dict(state_bits=16), "state_bits"), (dict(max_norm=0.0), "max_norm"), (dict(max_norm=math.nan), "max_norm"),
                      (dict(seed=2 ** 64), "seed"), (dict(lr=-1.0), "lr"), (dict(lr=math.nan), "lr"), (dict(betas=(1.0, 0.9)), "betas"),
                      (dict(betas=(0.9, -0.1)), "betas"), (dict(eps=0.0), "eps"), (dict(eps=1e-60), "eps"), (dict(eps=1e-40), "eps"),
                      (dict(weight_decay=-0.1), "weight_decay"), (dict(lr=torch.zeros(2, device="cuda")), "lr tensor"),
                      (dict(lr=torch.zeros(())), "lr tensor")):
        with pytest.raises(ValueError, match=match):
            optim.AdamW(**ok, **kw)
    with pytest.raises(TypeError, match="dtype"):
        optim.AdamW([torch.nn.Parameter(torch.zeros(3, device="cuda", dtype=torch.float64))])
    with pytest.raises(ValueError, match="CUDA"):
        optim.AdamW([torch.nn.Parameter(torch.zeros(3))])
    with pytest.raises(ValueError, match="gaps"):
        optim.AdamW([torch.nn.Parameter(torch.zeros(4, 4, device="cuda")[:, ::2])])
    with pytest.raises(ValueError, match="16 groups"):
        optim.AdamW([dict(params=[torch.nn.Parameter(torch.zeros(1, device="cuda"))]) for _ in range(17)])
    none = torch.nn.Parameter(torch.zeros(0, 3, device="cuda"))
    none.grad = torch.zeros(0, 3, device="cuda")
    opt = optim.AdamW([none], state_bits=8, max_norm=1.0)
    opt.step()
    assert int(opt.steps()) == 0 and opt.moments()[0].numel() == 0
    q = torch.zeros(20, device="cuda")
    opt = optim.AdamW([torch.nn.Parameter(q[:12]), torch.nn.Parameter(q[11:])])
    with pytest.raises(ValueError, match="share memory"):
        opt.step()
    opt = optim.AdamW([p])
    opt.step()  # no gradient at all: no step
    assert int(opt.steps()) == 0
    p.grad = torch.zeros(10, 10, device="cuda")
    opt.step()
    p.grad = None
    p.data = p.data.half()
    p.grad = torch.zeros(10, 10, device="cuda", dtype=FP16)
    with pytest.raises(ValueError, match="changed"):
        opt.step()
    p.grad = None
    p.data = torch.zeros(10, 10, device="cuda")
    p.grad = torch.sparse_coo_tensor(torch.zeros(2, 1, dtype=torch.long), torch.ones(1), (10, 10), device="cuda")
    with pytest.raises(TypeError, match="dense"):
        opt.step()
    assert int(opt.steps()) == 1

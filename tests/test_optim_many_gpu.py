"""8-bit averages over more tensors than a launch takes, and gradients of which many rows are zeros.  Codes are whole numbers
and equal the restatement's (oracle/step_ref.py)."""
import math

import numpy as np
import pytest
import torch

from oracle import step_ref as ref
from test_optim_gpu import E

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,master,max_norm", [(torch.float32, False, None), (torch.bfloat16, True, 2.0)])
def test_8_bit_averages_of_more_tensors_than_a_launch_takes(dtype, master, max_norm):
    from rl_for_mario_b200 import optim

    g = torch.Generator().manual_seed(7)
    sizes = [1 + i * 37 % 700 for i in range(1700)]  # 768, 768 and 164 tensors
    ps = [torch.nn.Parameter((torch.randn(n, generator=g) * 0.05).to(dtype).cuda()) for n in sizes]
    opt = optim.AdamW(ps, lr=1e-2, state_bits=8, master=master, max_norm=max_norm, seed=21)
    blocks = [(n + 255) // 256 for n in sizes]
    total = sum(blocks) * 256
    for t in (1, 2):
        xs = [(torch.randn(n, generator=g) * 1e-2).to(dtype) for n in sizes]
        for p, x in zip(ps, xs):
            p.grad = x.cuda()
        m0, v0 = (y.float().cpu().numpy() for y in opt.moments())
        old = opt.master.cpu() if master else torch.cat([torch.nn.functional.pad(p.detach().cpu(), (0, b * 256 - p.numel()))
                                                         for p, b in zip(ps, blocks)])
        opt.step()
        flat = torch.cat([torch.nn.functional.pad(x.float(), (0, b * 256 - len(x))) for x, b in zip(xs, blocks)])
        clip = None
        if max_norm is not None:
            norm = math.sqrt(flat.double().pow(2).sum().item())
            assert norm > max_norm and abs(opt.norm.item() - norm) <= norm * 5 * E
            clip = np.minimum(np.float32(1), np.float32(max_norm) / (np.float32(opt.norm.item()) + np.float32(1e-6)))
        m1, v1 = ref.averages_f32(m0, v0, flat.numpy(), 0.9, 0.999, clip)
        words = ref.step_words(total, 21, t)
        state = opt.state_dict()["state"]
        for name, y, w, kind in (("exp_avg", m1, words[0], ref.FIRST), ("exp_avg_sq", v1, words[1], ref.SECOND)):
            codes, scales = ref.encode(y, w, kind)
            assert np.array_equal(state[name].cpu().numpy(), codes)
            assert np.array_equal(state[name + "_scale"].cpu().numpy(), scales)
        r = ref.adamw(old, flat, torch.from_numpy(m0), torch.from_numpy(v0), t, 1e-2, 0.9, 0.999, 1e-8, 1e-2,
                      1.0 if clip is None else max_norm / (norm + 1e-6))
        want, (ap, au) = r["p"]
        tol = 4 * E * ap + 40 * E * au + E * want.abs()
        now = opt.master.cpu() if master else None
        at = 0
        for p, b in zip(ps, blocks):
            n = p.numel()
            got = (now[at:at + n] if master else p.detach().cpu()).double()
            assert ((got - want[at:at + n]).abs() <= tol[at:at + n]).all()
            if master:
                assert torch.equal(p.detach().cpu(), now[at:at + n].to(dtype))
            at += b * 256
    assert int(opt.steps()) == 2


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradients_of_zero_rows(dtype):
    """An embedding of which a batch used a few rows: the norm, and the step of rows with and without a gradient."""
    from rl_for_mario_b200 import optim

    g = torch.Generator().manual_seed(2)
    x = torch.randn(4096, 96, generator=g) * (torch.rand(4096, 1, generator=g) < 0.03)
    x = x.to(dtype)
    assert (x == 0).all(1).sum() > 3500
    want = math.sqrt(x.double().pow(2).sum().item())
    assert abs(optim.grad_norm([x.cuda()]).item() - want) <= want * 5 * E
    assert optim.grad_norm([torch.zeros(4096, 96, device="cuda", dtype=dtype)]).item() == 0
    for bits in (32, 8):
        p = torch.nn.Parameter(torch.ones(4096, 96, device="cuda", dtype=dtype))
        opt = optim.AdamW([p], lr=0.25, weight_decay=0.0, state_bits=bits, max_norm=1e9)
        p.grad = x.cuda()
        opt.step()
        # (No average is zero where the gradient is not; a first step is the rate, whatever the gradient's size.)
        moved = (p.detach().float().cpu() - 1).abs()
        assert (moved[x == 0] == 0).all() and ((moved[x != 0] - 0.25).abs() < 0.01).all()

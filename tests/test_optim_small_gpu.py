"""AdamW with an eps so small that averages below the normal numbers of fp32 count, in 8 and in 32 bits, against the float64
restatement.

Tolerances as in test_optim_gpu.py, with one more term: v' is a sum of two rounded products, one of them of a rounded
square, each off by up to 2^-150 where it is below the normal numbers: 2^-148 holds them, and moves the root, and with it the
step, by half of its part of v'.
"""
import math

import numpy as np
import pytest
import torch

from oracle import step_ref as ref
from test_optim_gpu import E, memory, near

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
pytestmark = pytest.mark.gpu

# eps sqrt(1 - beta2) against 2^-38 = 3.64e-12 decides on how the kernel takes 8-bit averages' roots: 1.151e-10 with 0.999.
CASES = [(1e-30, 0.999), (2e-38, 0.999), (1.14e-10, 0.999), (1.17e-10, 0.999), (1e-12, 0.0), (1e-8, 1 - 1e-9)]


@pytest.mark.parametrize("eps,b2", CASES)
@pytest.mark.parametrize("bits,dtype,master", [(8, FP32, False), (8, BF16, False), (8, BF16, True), (32, FP32, False)])
def test_averages_below_the_normal_numbers(bits, dtype, master, eps, b2):
    from rl_for_mario_b200 import optim

    n, b1, lr = 5003, 0.9, 1e-2
    g = torch.Generator().manual_seed(3)
    p = torch.nn.Parameter((torch.randn(n, generator=g) * 0.05).to(dtype).cuda())
    # Whole blocks of one size (their scale is their own), sizes from 1e-19 to 1; a block of zeros.
    size = torch.logspace(-19, 0, n // 256 + 1).repeat_interleave(256)[:n]
    size[1024:1280] = 0
    groups = [dict(params=[p]), dict(params=[torch.nn.Parameter(torch.ones(3, device="cuda"))], eps=1e-3, betas=(0.9, 0.99))]
    opt = optim.AdamW(groups, lr=lr, betas=(b1, b2), eps=eps, weight_decay=0.1, state_bits=bits, master=master, seed=5)
    for t in (1, 2, 3):
        x = (torch.randn(n, generator=g).abs() + 1).mul(torch.rand(n, generator=g).sub(0.5).sign()) * size
        p.grad = x.to(dtype).cuda()
        x = p.grad.cpu()
        m, v = (y[:n].float().cpu() for y in opt.moments())
        w = opt.master[:n].cpu() if master else memory(p).cpu()
        opt.step()
        r = ref.adamw(w, x, m, v, t, lr, b1, b2, eps, 0.1)
        want, (ap, au) = r["p"]
        v1 = r["v"][0]
        assert (v1[:256] > 0).all() and v1[:256].min() < 2.0 ** -126
        root = (v1 / (1 - b2 ** t)).sqrt()
        # (The root's part of the denominator moves by half of v's relative part.)
        moved = torch.where(v1 > 0, au * (2.0 ** -148 / 2 / v1.clamp(min=1e-44)) * root / (root + eps), torch.zeros(()).double())
        tol = 4 * E * ap + 40 * E * au + E * want.abs() + 1.1 * moved
        got = opt.master[:n] if master else memory(p)
        u = 0 if master or dtype == FP32 else torch.finfo(dtype).eps / 2
        near("p", got, want, tol * (1 + u) + u * want.abs())
        if t == 1 and eps < 1e-13:  # a step of the rate, whatever the gradient's size
            step = (want - w.double() * (1 - lr * 0.1)).abs()[size > 0]
            assert (step / lr - 1).abs().max() < 1e-2
    assert int(opt.steps()) == 3

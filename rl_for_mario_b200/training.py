"""Training operators as autograd functions, and the state of their dropout generator.

The reference trains this model with dropout (trainer/train_pretrain.py:121-129;
model/model_decision_transformer.py:153-163, :256-271, :420): ``attention`` /
``attention_qkv`` are the causal GQA attention with its gradient, ``qkv_rope``
the Q/K/V projection with RoPE and its gradient, ``head_norm_rope`` the norm of every
query and key head with the RoPE behind it (``attention_qk_norm``: with the attention
behind that), ``residual_norm`` the residual add with the norms before and after it, its gate and dropout, ``dropout`` the
plain one.  ``MarioDT.fuse_training()`` and ``FastDTAttention.fuse_training()``
run a model on them.

A dropout mask is a function of (seed, step, site, element) that the forward
and backward kernels evaluate; it is never stored.  ``DropoutState`` holds the
seed and the step on the device: ``draw()`` hands out the pair for one forward
pass and moves on, so passes have masks of their own, a backward pass sees the
pair of its forward pass whatever was drawn since, and a captured graph draws
anew at each replay.  ``site`` tells the places of a model apart.

What follows from that: ranks of a data-parallel job take seeds of their own; a
forward pass that is run again for its backward pass (activation checkpointing)
has to be given the first one's pair, since a new draw() is another mask; and a
state that two streams draw from at once is theirs to order.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import kernels

Tensor = torch.Tensor


class DropoutState:
    """Seed and step of the dropout generator on a device."""

    def __init__(self, seed: int, device="cuda"):
        if not -2 ** 63 <= int(seed) < 2 ** 64:
            raise ValueError("seed must fit 64 bits")
        seed = int(seed) - 2 ** 64 if int(seed) >= 2 ** 63 else int(seed)
        self.state = torch.tensor([seed, 0], dtype=torch.int64, device=device)

    def draw(self) -> Tensor:
        """(seed, step) for one forward pass, as a tensor of its own; the state moves to the next step."""
        now = self.state.clone()
        self.state[1:].add_(1)
        return now

    def to(self, device) -> "DropoutState":
        """The same seed and step, held on the device."""
        self.state = self.state.to(device)
        return self

    def state_dict(self) -> dict:
        seed, step = self.state.tolist()
        return {"seed": seed, "step": step}

    def load_state_dict(self, d: dict) -> None:
        self.state.copy_(torch.tensor([d["seed"], d["step"]], dtype=torch.int64))


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, pad_len, scale, p, rng, site):
        out, lse = kernels.attn_train_forward(q, k, v, pad_len, scale, p, rng, site)
        ctx.save_for_backward(q, k, v, out, lse, pad_len, rng)
        ctx.how = (scale, p, site)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse, pad_len, rng = ctx.saved_tensors
        scale, p, site = ctx.how
        dq, dk, dv = kernels.attn_train_backward(dout, q, k, v, out, lse, pad_len, scale, p, rng, site)
        return dq, dk, dv, None, None, None, None, None


def attention(q: Tensor, k: Tensor, v: Tensor, pad_len: Optional[Tensor] = None, scale: Optional[float] = None,
              p: float = 0.0, rng: Optional[Tensor] = None, site: int = 0) -> Tensor:
    """Differentiable causal GQA attention (kernels.attn_train_forward): q [B,S,Hq,D], k / v [B,S,Hkv,D]."""
    return _Attention.apply(q, k, v, pad_len, scale, p, rng, site)


class _AttentionQKV(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, heads, kv_heads, pad_len, scale, p, rng, site):
        q, k, v = qkv.split([heads, kv_heads, kv_heads], 2)
        out, lse = kernels.attn_train_forward(q, k, v, pad_len, scale, p, rng, site)
        ctx.save_for_backward(qkv, out, lse, pad_len, rng)
        ctx.how = (heads, kv_heads, scale, p, site)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        qkv, out, lse, pad_len, rng = ctx.saved_tensors
        heads, kv_heads, scale, p, site = ctx.how
        parts = [heads, kv_heads, kv_heads]
        dqkv = torch.empty(qkv.shape, dtype=qkv.dtype, device=qkv.device)
        kernels.attn_train_backward(dout, *qkv.split(parts, 2), out, lse, pad_len, scale, p, rng, site,
                                    grads=tuple(dqkv.split(parts, 2)))
        return dqkv, None, None, None, None, None, None, None


def attention_qkv(qkv: Tensor, heads: int, kv_heads: int, pad_len: Optional[Tensor] = None,
                  scale: Optional[float] = None, p: float = 0.0, rng: Optional[Tensor] = None,
                  site: int = 0) -> Tensor:
    """attention() on one projection output [B, S, heads + 2 kv_heads, D]; its gradient is written as one
    tensor of that shape, without a pass to put the three together."""
    if qkv.dim() != 4 or qkv.shape[2] != heads + 2 * kv_heads:
        raise ValueError(f"qkv must be [B, S, {heads + 2 * kv_heads}, D] (got {tuple(qkv.shape)})")
    return _AttentionQKV.apply(qkv, heads, kv_heads, pad_len, scale, p, rng, site)


class _QKVRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, cos, sin, rope_cols, head_dim):
        ctx.save_for_backward(x, w, cos, sin)
        ctx.how = (rope_cols, head_dim)
        return kernels.qkv_rope(x, w, cos, sin, rope_cols, head_dim)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, w, cos, sin = ctx.saved_tensors
        # The incoming gradient may be shared with other uses of y: rotate a tensor of this call's own.
        g = kernels.rope_grad_(dy.clone(memory_format=torch.contiguous_format), cos, sin, *ctx.how)
        g2 = g.view(-1, g.shape[-1])
        dx = (g2 @ w).view(x.shape) if ctx.needs_input_grad[0] else None
        dw = g2.t() @ x.reshape(-1, x.shape[-1]) if ctx.needs_input_grad[1] else None
        return dx, dw, None, None, None, None


def qkv_rope(x: Tensor, w: Tensor, cos: Tensor, sin: Tensor, rope_cols: int, head_dim: int) -> Tensor:
    """Differentiable kernels.qkv_rope: x [B, S, K] @ w^T with the RoPE of its first rope_cols columns."""
    return _QKVRope.apply(x, w, cos, sin, rope_cols, head_dim)


class _HeadNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, eps, cos, sin, start_pos):
        ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin, start_pos)
        ctx.eps = eps
        return kernels.head_norm_rope_forward(q, k, q_weight, k_weight, eps, cos, sin, start_pos)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq_out, dk_out):
        q, k, q_weight, k_weight, cos, sin, start_pos = ctx.saved_tensors
        dq, dk, dwq, dwk = kernels.head_norm_rope_backward(dq_out, dk_out, q, k, q_weight, k_weight, ctx.eps, cos, sin,
                                                           start_pos)
        return dq, dk, dwq, dwk, None, None, None, None


def head_norm_rope(q: Tensor, k: Tensor, q_weight: Tensor, k_weight: Tensor, eps: float, cos: Tensor, sin: Tensor,
                   start_pos: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
    """Differentiable kernels.head_norm_rope_forward: q [B,S,Hq,D] and k [B,S,Hkv,D] with every head normalised and
    rotated."""
    return _HeadNormRope.apply(q, k, q_weight, k_weight, eps, cos, sin, start_pos)


class _AttentionQKNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, q_weight, k_weight, heads, kv_heads, eps, cos, sin, pad_len, scale, p, rng, site):
        q, k, v = qkv.split([heads, kv_heads, kv_heads], 2)
        q, k = kernels.head_norm_rope_forward(q, k, q_weight, k_weight, eps, cos, sin)
        out, lse = kernels.attn_train_forward(q, k, v, pad_len, scale, p, rng, site)
        ctx.save_for_backward(qkv, q, k, q_weight, k_weight, cos, sin, out, lse, pad_len, rng)
        ctx.how = (heads, kv_heads, eps, scale, p, site)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        qkv, q, k, q_weight, k_weight, cos, sin, out, lse, pad_len, rng = ctx.saved_tensors
        heads, kv_heads, eps, scale, p, site = ctx.how
        parts = [heads, kv_heads, kv_heads]
        xq, xk, v = qkv.split(parts, 2)
        dqkv = torch.empty(qkv.shape, dtype=qkv.dtype, device=qkv.device)
        dq, dk, dv = dqkv.split(parts, 2)
        kernels.attn_train_backward(dout, q, k, v, out, lse, pad_len, scale, p, rng, site, grads=(dq, dk, dv))
        _, _, dwq, dwk = kernels.head_norm_rope_backward(dq, dk, xq, xk, q_weight, k_weight, eps, cos, sin,
                                                         grads=(dq, dk))
        return dqkv, dwq, dwk, None, None, None, None, None, None, None, None, None, None


def attention_qk_norm(qkv: Tensor, heads: int, kv_heads: int, q_weight: Tensor, k_weight: Tensor, eps: float,
                      cos: Tensor, sin: Tensor, pad_len: Optional[Tensor] = None, scale: Optional[float] = None,
                      p: float = 0.0, rng: Optional[Tensor] = None, site: int = 0) -> Tensor:
    """attention_qkv() on a projection output whose query and key heads are normalised and rotated first (rows 0 .. S - 1
    of the tables); the gradient of the projection is written as one tensor, the heads' in place."""
    if qkv.dim() != 4 or qkv.shape[2] != heads + 2 * kv_heads:
        raise ValueError(f"qkv must be [B, S, {heads + 2 * kv_heads}, D] (got {tuple(qkv.shape)})")
    return _AttentionQKNorm.apply(qkv, q_weight, k_weight, heads, kv_heads, eps, cos, sin, pad_len, scale, p, rng, site)


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, pre_weight, post_weight, gate, eps, alpha, p, rng, site):
        h, n, stats = kernels.residual_norm_forward(x, residual, pre_weight, eps, post_weight, gate, alpha, p, rng,
                                                    site)
        ctx.save_for_backward(x, residual, pre_weight, post_weight, gate, stats, rng)
        ctx.how = (alpha, p, site)
        ctx.set_materialize_grads(False)  # an output without a gradient is read as zero by the kernel
        return h, n

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh, dn):
        x, residual, pre_weight, post_weight, gate, stats, rng = ctx.saved_tensors
        alpha, p, site = ctx.how
        dx, dres, dpre, dpost, dgate = kernels.residual_norm_backward(dh, dn, x, residual, pre_weight, stats,
                                                                      post_weight, gate, alpha, p, rng, site)
        return dx, None if residual is None else dres, dpre, dpost, dgate, None, None, None, None, None


def residual_norm(x: Tensor, residual: Optional[Tensor], pre_weight: Tensor, eps: float,
                  post_weight: Optional[Tensor] = None, gate: Optional[Tensor] = None, alpha: float = 1.0,
                  p: float = 0.0, rng: Optional[Tensor] = None, site: int = 0) -> Tuple[Tensor, Tensor]:
    """Differentiable kernels.residual_norm_forward: (h, n) with
    h = residual + alpha * gate * dropout(RMSNorm(x) * post_weight), n = RMSNorm(h) * pre_weight."""
    return _ResidualNorm.apply(x, residual, pre_weight, post_weight, gate, eps, alpha, p, rng, site)


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, rng, site):
        ctx.save_for_backward(rng)
        ctx.how = (p, site)
        return kernels.dropout_forward(x, p, rng, site, residual)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        p, site = ctx.how
        dx = kernels.dropout_backward(dy, p, ctx.saved_tensors[0], site) if ctx.needs_input_grad[0] else None
        return dx, dy if ctx.needs_input_grad[1] else None, None, None, None


def dropout(x: Tensor, p: float, rng: Optional[Tensor], site: int = 0, residual: Optional[Tensor] = None) -> Tensor:
    """Differentiable kernels.dropout_forward: residual + dropout(x)."""
    return _Dropout.apply(x, residual, p, rng, site)

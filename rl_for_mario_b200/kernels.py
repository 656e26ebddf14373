"""Tensor-level wrappers over the C-ABI entry points.

Each wrapper validates device / dtype, allocates its outputs with torch (the
library itself never allocates), and launches on torch's current CUDA stream.
"""
from __future__ import annotations

import ctypes
import functools
import math
import struct
from typing import Optional, Tuple

import torch

from . import _lib

Tensor = torch.Tensor

_DTYPES = {torch.bfloat16: _lib.DT_DTYPE_BF16, torch.float16: _lib.DT_DTYPE_FP16,
           torch.float32: _lib.DT_DTYPE_FP32}


def _dtype_code(t: Tensor) -> int:
    try:
        return _DTYPES[t.dtype]
    except KeyError:
        raise TypeError(f"unsupported dtype {t.dtype}") from None


# torch's own shortcuts past the objects of current_stream() and current_device() (a microsecond a call), where this
# torch has them.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_raw_device = getattr(torch._C, "_cuda_getDevice", None)


def _stream_ptr(device: torch.device) -> int:
    if _raw_stream is None or device.index is None:
        return torch.cuda.current_stream(device).cuda_stream
    return _raw_stream(device.index)


def _ptr(t: Optional[Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _require_cuda(*ts: Optional[Tensor]) -> None:
    for t in ts:
        if t is not None and not t.is_cuda:
            raise ValueError("dt attention kernels take CUDA tensors only (no CPU path)")


def _rope_mode(apply_rope) -> int:
    """apply_rope of the entry points: False / 0 none, True / 1 RoPE in fp32 with one
    rounding of the result, 2 the reference's roundings in the activation dtype
    (q * cos, rotate_half(q) * sin and their sum each rounded, as on 16-bit tensors)."""
    mode = int(apply_rope)
    if mode not in (0, 1, 2):
        raise ValueError(f"apply_rope must be False/True or 0, 1, 2 (got {apply_rope!r})")
    return mode


def pad_len_from_mask(attention_mask: Tensor, S: int) -> Tensor:
    """Left-padding length per row of a [B, S] 0/1 mask (1 = valid), as int32 on its device.

    The DT dataset left-pads (scripts/mario/dt_offline_dataset.py:228-235), so
    the number of zeros is the index of the first valid token.
    """
    m = attention_mask.reshape(attention_mask.shape[0], -1)
    if m.shape[1] != S:
        raise ValueError(f"attention_mask has {m.shape[1]} columns, expected {S}")
    return (S - (m != 0).sum(dim=1)).to(torch.int32)


def attn_prefill(q: Tensor, k: Tensor, v: Tensor, cos: Optional[Tensor], sin: Optional[Tensor],
                 pad_len: Optional[Tensor] = None, out: Optional[Tensor] = None, apply_rope: bool = True,
                 scale: Optional[float] = None) -> Tensor:
    """Causal GQA prefill: q [B,S,Hq,D], k/v [B,S,Hkv,D] -> out [B,S,Hq,D].

    RoPE (cos/sin [>=S, D] fp32) is applied to q and k inside the kernel when
    apply_rope (2: with the reference's roundings, see _rope_mode); pad_len [B]
    int32 gives per-row left padding (None = no mask).
    """
    _require_cuda(q, k, v, cos, sin, pad_len, out)
    B, S, Hq, D = q.shape
    Hkv = k.shape[2]
    if k.shape != (B, S, Hkv, D) or v.shape != (B, S, Hkv, D):
        raise ValueError(f"k/v shapes {tuple(k.shape)}, {tuple(v.shape)} do not match q {tuple(q.shape)}")
    if not (q.dtype == k.dtype == v.dtype):
        raise TypeError("q, k, v must share a dtype")
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.stride(3) != 1:
            raise ValueError(f"{name} must be contiguous in head_dim")
    if out is None:
        out = torch.empty((B, S, Hq, D), dtype=q.dtype, device=q.device)
    if apply_rope:
        if cos is None or sin is None:
            raise ValueError("apply_rope needs cos and sin")
        cos = cos.float().contiguous() if (cos.dtype != torch.float32 or cos.stride(-1) != 1) else cos
        sin = sin.float().contiguous() if (sin.dtype != torch.float32 or sin.stride(-1) != 1) else sin
        if cos.stride(0) != sin.stride(0):
            cos, sin = cos.contiguous(), sin.contiguous()
    if pad_len is not None:
        pad_len = pad_len.to(torch.int32).contiguous()
    lib = _lib.load()
    rc = lib.dt_attn_prefill(
        _ptr(q), _ptr(k), _ptr(v), _ptr(out), _ptr(cos) if apply_rope else None,
        _ptr(sin) if apply_rope else None, cos.shape[0] if apply_rope else 0,
        cos.stride(0) if apply_rope else 0, _ptr(pad_len), B, S, Hq, Hkv, D,
        q.stride(0), q.stride(1), q.stride(2), k.stride(0), k.stride(1), k.stride(2),
        v.stride(0), v.stride(1), v.stride(2), out.stride(0), out.stride(1), out.stride(2),
        float(scale) if scale is not None else 0.0, _rope_mode(apply_rope), _dtype_code(q),
        _stream_ptr(q.device))
    _lib.check("dt_attn_prefill", rc)
    return out


_COPY_STREAMS: dict = {}


def _copy_streams(device: torch.device):
    """A host-to-device and a device-to-host stream per device (created once)."""
    key = device.index if device.index is not None else torch.cuda.current_device()
    if key not in _COPY_STREAMS:
        _COPY_STREAMS[key] = (torch.cuda.Stream(device=key), torch.cuda.Stream(device=key))
    return _COPY_STREAMS[key]


def attn_prefill_host(hq: Tensor, hk: Tensor, hv: Tensor, cos: Optional[Tensor], sin: Optional[Tensor],
                      hpad: Optional[Tensor], hout: Tensor, device_buffers: Tuple[Tensor, ...],
                      chunks: int = 8, apply_rope: bool = True, scale: Optional[float] = None) -> Tensor:
    """attn_prefill on host tensors: q/k/v (and pad_len) in pinned host memory in,
    out into the pinned host tensor ``hout``.

    The batch is cut into ``chunks`` pieces of whole samples (samples are
    independent) and pipelined over three streams: the copy of chunk i + 1 to
    the device, the kernel on chunk i (current stream) and the copy of chunk
    i - 1 back run at the same time, so the step costs about the larger of the
    two PCIe transfers instead of their sum.  ``device_buffers`` = (q, k, v,
    pad_len or None, out) device tensors of the full batch's shapes.  On return
    the current stream is ordered after every copy (synchronise it, or record an
    event on it, before reading ``hout`` on the host).
    """
    dq, dk, dv, dpad, dout = device_buffers
    for name, h in (("hq", hq), ("hk", hk), ("hv", hv), ("hout", hout), ("hpad", hpad)):
        if h is not None and (h.is_cuda or not h.is_pinned()):
            raise ValueError(f"{name} must be a pinned host tensor")
    _require_cuda(dq, dk, dv, dpad, dout)
    if (hpad is None) != (dpad is None):
        raise ValueError("hpad and the device pad_len buffer go together")
    # Tensor.copy_ would silently cast or broadcast: host and device buffers
    # must match exactly.
    for name, h, d in (("q", hq, dq), ("k", hk, dk), ("v", hv, dv), ("out", hout, dout), ("pad_len", hpad, dpad)):
        if h is not None and (h.dtype != d.dtype or h.shape != d.shape):
            raise ValueError(f"host {name} {tuple(h.shape)} {h.dtype} does not match its device buffer "
                             f"{tuple(d.shape)} {d.dtype}")
    B = hq.shape[0]
    chunks = max(1, min(int(chunks), B))
    bounds = [B * i // chunks for i in range(chunks + 1)]
    dev = dq.device
    cur = torch.cuda.current_stream(dev)
    s_in, s_out = _copy_streams(dev)
    # Earlier work on the current stream (a previous call's kernels reading these
    # buffers) comes before this call's uploads.
    s_in.wait_stream(cur)
    for i in range(chunks):
        b0, b1 = bounds[i], bounds[i + 1]
        if b1 == b0:
            continue
        with torch.cuda.stream(s_in):
            dq[b0:b1].copy_(hq[b0:b1], non_blocking=True)
            dk[b0:b1].copy_(hk[b0:b1], non_blocking=True)
            dv[b0:b1].copy_(hv[b0:b1], non_blocking=True)
            if hpad is not None:
                dpad[b0:b1].copy_(hpad[b0:b1], non_blocking=True)
        cur.wait_stream(s_in)
        attn_prefill(dq[b0:b1], dk[b0:b1], dv[b0:b1], cos, sin, None if dpad is None else dpad[b0:b1],
                     out=dout[b0:b1], apply_rope=apply_rope, scale=scale)
        s_out.wait_stream(cur)
        with torch.cuda.stream(s_out):
            hout[b0:b1].copy_(dout[b0:b1], non_blocking=True)
    cur.wait_stream(s_out)
    return hout


def device_status(device: Optional[torch.device] = None) -> int:
    """Synchronises the current stream; returns and clears the kernels' device status word."""
    dev = device or torch.device("cuda", torch.cuda.current_device())
    return _lib.load().dt_device_status(_stream_ptr(dev))


def default_scale(D: int) -> float:
    return 1.0 / math.sqrt(D)


def _prep_tables(cos: Optional[Tensor], sin: Optional[Tensor]):
    if cos is None or sin is None:
        raise ValueError("apply_rope needs cos and sin")
    if cos.dtype != torch.float32 or cos.stride(-1) != 1:
        cos = cos.float().contiguous()
    if sin.dtype != torch.float32 or sin.stride(-1) != 1:
        sin = sin.float().contiguous()
    if cos.stride(0) != sin.stride(0):
        cos, sin = cos.contiguous(), sin.contiguous()
    return cos, sin


def attn_decode(q: Tensor, k_new: Tensor, v_new: Tensor, layer, cos: Optional[Tensor], sin: Optional[Tensor],
                pad_len: Optional[Tensor] = None, rope_abs: bool = False, out: Optional[Tensor] = None,
                apply_rope: bool = True, scale: Optional[float] = None) -> Tensor:
    """Cached decode step: q [B,Sn,Hq,D], k_new/v_new [B,Sn,Hkv,D] -> out [B,Sn,Hq,D].

    Appends the rotated k_new / v_new to ``layer`` (a cache.LayerKV) at
    positions layer.seq_lens .. +Sn and attends over all cached keys.  Does not
    advance the layer's length (the caller does, once per step).
    """
    _require_cuda(q, k_new, v_new, cos, sin, pad_len, out)
    B, Sn, Hq, D = q.shape
    Hkv = k_new.shape[2]
    if k_new.shape != (B, Sn, Hkv, D) or v_new.shape != (B, Sn, Hkv, D):
        raise ValueError("k_new/v_new shapes do not match q")
    if not (q.dtype == k_new.dtype == v_new.dtype == layer.k_pages.dtype):
        raise TypeError("q, k_new, v_new and the cache must share a dtype")
    if layer.batch != B or layer.num_kv_heads != Hkv or layer.head_dim != D:
        raise ValueError("cache geometry does not match the inputs")
    if layer.length + Sn > layer.capacity:
        raise ValueError(f"cache full: {layer.length} + {Sn} > capacity {layer.capacity}")
    for name, t in (("q", q), ("k_new", k_new), ("v_new", v_new)):
        if t.stride(3) != 1:
            raise ValueError(f"{name} must be contiguous in head_dim")
    if out is None:
        out = torch.empty((B, Sn, Hq, D), dtype=q.dtype, device=q.device)
    if apply_rope:
        cos, sin = _prep_tables(cos, sin)
    if pad_len is not None:
        pad_len = pad_len.to(torch.int32).contiguous()
    lib = _lib.load()
    rc = lib.dt_attn_decode(
        _ptr(q), _ptr(k_new), _ptr(v_new), _ptr(out), _ptr(layer.k_pages), _ptr(layer.v_pages),
        layer.k_pages.shape[0], layer.page_size, _ptr(layer.block_table), layer.block_table.shape[1],
        _ptr(layer.seq_lens), _ptr(pad_len), _ptr(cos) if apply_rope else None, _ptr(sin) if apply_rope else None,
        cos.shape[0] if apply_rope else 0, cos.stride(0) if apply_rope else 0, 1 if rope_abs else 0,
        B, Sn, Hq, Hkv, D, q.stride(0), q.stride(1), q.stride(2), k_new.stride(0), k_new.stride(1),
        k_new.stride(2), v_new.stride(0), v_new.stride(1), v_new.stride(2), out.stride(0), out.stride(1),
        out.stride(2), float(scale) if scale is not None else 0.0, _rope_mode(apply_rope), _dtype_code(q),
        _stream_ptr(q.device))
    _lib.check("dt_attn_decode", rc)
    return out


def kv_write(k: Tensor, v: Tensor, layer, cos: Optional[Tensor], sin: Optional[Tensor],
             start_pos: Optional[Tensor] = None, rope_abs: bool = False, apply_rope: bool = True) -> None:
    """Writes k (rotated) and v [B,S,Hkv,D] into ``layer`` at positions start_pos[b] + s."""
    _require_cuda(k, v, cos, sin, start_pos)
    B, S, Hkv, D = k.shape
    if v.shape != k.shape:
        raise ValueError("k and v shapes differ")
    if k.dtype != layer.k_pages.dtype or v.dtype != k.dtype:
        raise TypeError("k, v and the cache must share a dtype")
    if k.stride(3) != 1 or v.stride(3) != 1:
        raise ValueError("k/v must be contiguous in head_dim")
    if apply_rope:
        cos, sin = _prep_tables(cos, sin)
    if start_pos is not None:
        start_pos = start_pos.to(torch.int32).contiguous()
    lib = _lib.load()
    rc = lib.dt_kv_write(
        _ptr(k), _ptr(v), _ptr(layer.k_pages), _ptr(layer.v_pages), layer.k_pages.shape[0], layer.page_size,
        _ptr(layer.block_table), layer.block_table.shape[1], _ptr(start_pos), _ptr(cos) if apply_rope else None,
        _ptr(sin) if apply_rope else None, cos.shape[0] if apply_rope else 0, cos.stride(0) if apply_rope else 0,
        1 if rope_abs else 0, B, S, Hkv, D, k.stride(0), k.stride(1), k.stride(2), v.stride(0), v.stride(1),
        v.stride(2), _rope_mode(apply_rope), _dtype_code(k), _stream_ptr(k.device))
    _lib.check("dt_kv_write", rc)


def fold_norm_weight(w_q: Tensor, w_k: Tensor, w_v: Tensor, w_norm: Tensor, dtype: torch.dtype) -> Tensor:
    """[Wq; Wk; Wv] * diag(w_norm) in ``dtype``: the weight of rmsnorm_qkv."""
    w = torch.cat([w_q, w_k, w_v], dim=0).float() * w_norm.float()[None, :]
    return w.to(dtype).contiguous()


def frames_to_blocks(frames: Tensor, dtype: torch.dtype, frame_max: Optional[Tensor] = None) -> Tensor:
    """uint8 frames [N, C, H, W] -> ``dtype`` 4 x 4 space-to-depth blocks as a
    channels-last [N, C*16, H/4, W/4] tensor (channel c*16 + dy*4 + dx).
    ``frame_max`` (an int32 [1] device tensor) is raised to the largest byte."""
    _require_cuda(frames, frame_max)
    if frame_max is not None and (frame_max.dtype != torch.int32 or frame_max.numel() != 1):
        raise ValueError("frame_max must be an int32 tensor with one element")
    if frames.dtype != torch.uint8 or frames.dim() != 4 or not frames.is_contiguous():
        raise ValueError("frames must be a contiguous uint8 [N, C, H, W] tensor")
    N, C, H, W = frames.shape
    out = torch.empty((N, C * 16, H // 4, W // 4), dtype=dtype, device=frames.device,
                      memory_format=torch.channels_last)
    rc = _lib.load().dt_frames_to_blocks(_ptr(frames), _ptr(out), N, C, H, W,
                                         None if frame_max is None else _ptr(frame_max), _dtype_code(out),
                                         _stream_ptr(frames.device))
    _lib.check("dt_frames_to_blocks", rc)
    return out


def frames_conv1(frames: Tensor, weight: Tensor, bias: Tensor, round_input: bool = False) -> Tuple[Tensor, Tensor]:
    """relu(conv2d(frames / 255 if max > 1 else frames, weight, bias, stride 4)) from
    uint8 frames [N, 4, H, W] with an 8 x 8 weight [32, 4, 8, 8] (16-bit): returns the
    output as a channels-last [N, 32, OH, OW] tensor of the weight's dtype and an
    int32 [1] device tensor that is > 1 exactly when the frames' max exceeds 1.
    round_input: frames / 255 rounded to the weight's dtype before the
    convolution (the reference's 16-bit rounding) instead of exact pixels."""
    _require_cuda(frames, weight, bias)
    if frames.dtype != torch.uint8 or frames.dim() != 4 or not frames.is_contiguous():
        raise ValueError("frames must be a contiguous uint8 [N, C, H, W] tensor")
    N, C, H, W = frames.shape
    if tuple(weight.shape) != (32, C, 8, 8):
        raise ValueError(f"weight must be [32, {C}, 8, 8]")
    OH, OW = (H - 8) // 4 + 1, (W - 8) // 4 + 1
    w2 = weight.reshape(32, C * 64).contiguous()
    b = bias.float().contiguous()
    out = torch.empty((N, 32, OH, OW), dtype=weight.dtype, device=frames.device, memory_format=torch.channels_last)
    fmax = torch.empty(1, dtype=torch.int32, device=frames.device)
    rc = _lib.load().dt_frames_conv1(_ptr(frames), N, C, H, W, _ptr(w2), _ptr(b), _ptr(fmax), _ptr(out),
                                     1 if round_input else 0, _dtype_code(out), _stream_ptr(frames.device))
    _lib.check("dt_frames_conv1", rc)
    return out, fmax


def encoder_conv23(x1: Tensor, w2: Tensor, b2: Tensor, w3: Tensor, b3: Tensor,
                   keep_y2: bool = True) -> Tuple[Optional[Tensor], Tensor]:
    """relu(conv2d(x1, w2, b2, stride 2)) and relu(conv2d(that, w3, b3)) for the
    state encoder's second and third layers: x1 a channels-last [N, 32, 20, 20]
    16-bit tensor (the first layer's output), w2 [64, 32, 4, 4], w3 [64, 64, 3, 3]
    of x1's dtype.  Returns both outputs as channels-last tensors ([N, 64, 9, 9],
    [N, 64, 7, 7]); with keep_y2=False the second layer's output is not written
    to memory at all (None is returned in its place)."""
    _require_cuda(x1, w2, b2, w3, b3)
    if x1.dim() != 4 or tuple(x1.shape[1:]) != (32, 20, 20) or not x1.is_contiguous(memory_format=torch.channels_last):
        raise ValueError("x1 must be a channels-last [N, 32, 20, 20] tensor")
    if tuple(w2.shape) != (64, 32, 4, 4) or tuple(w3.shape) != (64, 64, 3, 3):
        raise ValueError("w2 must be [64, 32, 4, 4] and w3 [64, 64, 3, 3]")
    if w2.dtype != x1.dtype or w3.dtype != x1.dtype or tuple(b2.shape) != (64,) or tuple(b3.shape) != (64,):
        raise ValueError("weights must have x1's dtype and biases 64 entries")
    N = x1.shape[0]
    w2c, w3c = w2.contiguous(), w3.contiguous()
    b2f, b3f = b2.float().contiguous(), b3.float().contiguous()
    cl = torch.channels_last
    y2 = torch.empty((N, 64, 9, 9), dtype=x1.dtype, device=x1.device, memory_format=cl) if keep_y2 else None
    y3 = torch.empty((N, 64, 7, 7), dtype=x1.dtype, device=x1.device, memory_format=cl)
    rc = _lib.load().dt_encoder_conv23(_ptr(x1), N, _ptr(w2c), _ptr(b2f), _ptr(y2), _ptr(w3c), _ptr(b3f), _ptr(y3),
                                       _dtype_code(x1), _stream_ptr(x1.device))
    _lib.check("dt_encoder_conv23", rc)
    return y2, y3


def rmsnorm(x: Tensor, weight: Tensor, eps: float, out: Optional[Tensor] = None) -> Tensor:
    """weight * cast(x * rsqrt(mean(x^2) + eps)) over the last dim (bf16 / fp16)."""
    _require_cuda(x, weight, out)
    K = x.shape[-1]
    if weight.shape != (K,) or weight.dtype != x.dtype or not weight.is_contiguous():
        raise ValueError("weight must be a contiguous [K] tensor of x's dtype")
    x2 = x.reshape(-1, K)
    if x2.stride(1) != 1:
        x2 = x2.contiguous()
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    o2 = out.view(-1, K)
    rc = _lib.load().dt_rmsnorm(_ptr(x2), x2.stride(0), _ptr(weight), _ptr(o2), o2.stride(0), x2.shape[0], K,
                                float(eps), _dtype_code(x), _stream_ptr(x.device))
    _lib.check("dt_rmsnorm", rc)
    return out


def fold_swiglu_weight(w_gate: Tensor, w_up: Tensor, w_norm: Tensor, dtype: torch.dtype) -> Tensor:
    """The weight of rmsnorm_swiglu: gate and up rows scaled by the norm weight,
    interleaved in blocks of 64 rows ([gate 0:64; up 0:64; gate 64:128; ...])."""
    inter, hidden = w_gate.shape
    if w_up.shape != w_gate.shape or inter % 64:
        raise ValueError("gate / up weights must be equal [F, H] with F a multiple of 64")
    nw = w_norm.float()[None, None, :]
    g = w_gate.float().view(inter // 64, 64, hidden) * nw
    u = w_up.float().view(inter // 64, 64, hidden) * nw
    return torch.stack((g, u), dim=1).reshape(2 * inter, hidden).to(dtype).contiguous()


def rmsnorm_swiglu(x: Tensor, w_fused: Tensor, eps: float, out: Optional[Tensor] = None) -> Tensor:
    """silu(g) * u with [g | u] = RMSNorm(x) @ [W_gate; W_up]^T: the post-attention
    norm and the SwiGLU up-projection of the block's MLP in one kernel.

    x [..., K] bf16/fp16 -> y [..., F], ``w_fused`` = fold_swiglu_weight(...) [2F, K].
    """
    _require_cuda(x, w_fused, out)
    K = x.shape[-1]
    F2 = w_fused.shape[0]
    if w_fused.shape[1] != K or w_fused.dtype != x.dtype or not w_fused.is_contiguous() or F2 % 128:
        raise ValueError("w_fused must be a contiguous [2F, K] tensor of x's dtype (F a multiple of 64)")
    x2 = x.reshape(-1, K)
    if x2.stride(1) != 1:
        x2 = x2.contiguous()
    M = x2.shape[0]
    if out is None:
        out = torch.empty(x.shape[:-1] + (F2 // 2,), dtype=x.dtype, device=x.device)
    o2 = out.view(-1, F2 // 2)
    rc = _lib.load().dt_rmsnorm_swiglu(_ptr(x2), x2.stride(0), _ptr(w_fused), _ptr(o2), o2.stride(0), M, K,
                                       F2 // 2, float(eps), _dtype_code(x), _stream_ptr(x.device))
    _lib.check("dt_rmsnorm_swiglu", rc)
    return out


def qkv_rope(x: Tensor, w_cat: Tensor, cos: Tensor, sin: Tensor, rope_cols: int, head_dim: int,
             out: Optional[Tensor] = None) -> Tensor:
    """[q | k | v] = x @ w_cat^T with the rotate-half RoPE of the q and k heads
    (the first rope_cols columns) in the GEMM epilogue, no norm: x [B, S, K]
    16-bit, w_cat = [Wq; Wk; Wv] [N, K] -> y [B, S, N]; row (b, s) uses table
    row s of cos / sin."""
    _require_cuda(x, w_cat, cos, sin, out)
    if x.dim() != 3:
        raise ValueError("qkv_rope needs x of shape [B, S, K]")
    K = x.shape[-1]
    N = w_cat.shape[0]
    if w_cat.shape[1] != K or w_cat.dtype != x.dtype or not w_cat.is_contiguous():
        raise ValueError("w_cat must be a contiguous [N, K] tensor of x's dtype")
    x2 = x.reshape(-1, K)
    if x2.stride(1) != 1:
        x2 = x2.contiguous()
    if out is None:
        out = torch.empty(x.shape[:-1] + (N,), dtype=x.dtype, device=x.device)
    o2 = out.view(-1, N)
    cos, sin = _prep_tables(cos, sin)
    rc = _lib.load().dt_qkv_rope(_ptr(x2), x2.stride(0), _ptr(w_cat), _ptr(o2), o2.stride(0), x2.shape[0], K, N,
                                 _ptr(cos), _ptr(sin), cos.stride(0), cos.shape[0], x.shape[1], int(rope_cols),
                                 int(head_dim), _dtype_code(x), _stream_ptr(x.device))
    _lib.check("dt_qkv_rope", rc)
    return out


def gemm_residual_ok(x: Tensor, w: Tensor, y: Tensor) -> bool:
    """Whether gemm_residual takes these operands (16-bit CUDA tensors, row-major
    views with 16-byte aligned rows, N a multiple of 64)."""
    if not (x.is_cuda and y.is_cuda and w.is_cuda):
        return False
    if x.dtype not in (torch.bfloat16, torch.float16) or w.dtype != x.dtype or y.dtype != x.dtype:
        return False
    K, N = x.shape[-1], y.shape[-1]
    if w.shape != (N, K) or N % 64 or K % 8 or not w.is_contiguous():
        return False
    for t in (x, y):
        if t.dim() != 2 or t.stride(1) != 1 or t.stride(0) % 8 or t.data_ptr() % 16:
            return False
    return x.shape[0] == y.shape[0]


_NUM_SMS: dict = {}


def gemm_residual_on_pairs(x: Tensor, w: Tensor, y: Tensor) -> bool:
    """Whether gemm_residual runs these operands on CTA pairs: N a multiple of 256 and
    at least four 256 x 256 tiles per pair of SMs, the sizes at which it matches
    cuBLAS's addmm (cfg4's o_proj / down_proj, measured).  Smaller, latency-bound
    problems (a rollout step's GEMMs) fall to the single-CTA kernel, which is slower
    than cuBLAS there."""
    if not gemm_residual_ok(x, w, y):
        return False
    M, N = y.shape
    dev = y.device.index if y.device.index is not None else torch.cuda.current_device()
    if dev not in _NUM_SMS:
        _NUM_SMS[dev] = torch.cuda.get_device_properties(dev).multi_processor_count
    return N % 256 == 0 and ((M + 255) // 256) * (N // 256) >= 2 * _NUM_SMS[dev]


def gemm_residual(x: Tensor, w: Tensor, y: Tensor) -> Tensor:
    """y += x @ w^T in place (fp32 accumulation, one rounding of the sum): the
    block's o_proj / down_proj with its residual add.  x [M, K], w [N, K],
    y [M, N] (2-D row-major views), bf16 / fp16."""
    _require_cuda(x, w, y)
    if not gemm_residual_ok(x, w, y):
        raise ValueError("gemm_residual: x [M, K], w [N, K] contiguous, y [M, N] 16-bit row-major views with "
                         "16-byte aligned rows and N a multiple of 64")
    rc = _lib.load().dt_gemm_residual(_ptr(x), x.stride(0), _ptr(w), _ptr(y), y.stride(0), x.shape[0], x.shape[1],
                                      y.shape[1], _dtype_code(x), _stream_ptr(x.device))
    _lib.check("dt_gemm_residual", rc)
    return y


def rmsnorm_qkv(x: Tensor, w_fused: Tensor, eps: float, out: Optional[Tensor] = None,
                rope: Optional[Tuple[Tensor, Tensor, int, int]] = None) -> Tensor:
    """y = RMSNorm(x) @ [Wq; Wk; Wv]^T with the norm weight folded into ``w_fused`` [N, K].

    x [..., K] bf16/fp16 (last dim contiguous) -> y [..., N] (the fused q|k|v rows).
    ``rope = (cos, sin, rope_cols, head_dim)`` also rotates the first rope_cols
    columns (the q and k heads) in the epilogue; x is then [B, S, K] and row
    (b, s) uses table row s.
    """
    _require_cuda(x, w_fused, out)
    if rope is not None:
        _require_cuda(rope[0], rope[1])
    K = x.shape[-1]
    N = w_fused.shape[0]
    if w_fused.shape[1] != K or w_fused.dtype != x.dtype or not w_fused.is_contiguous():
        raise ValueError("w_fused must be a contiguous [N, K] tensor of x's dtype")
    x2 = x.reshape(-1, K)
    if x2.stride(1) != 1:
        x2 = x2.contiguous()
    M = x2.shape[0]
    if out is None:
        out = torch.empty(x.shape[:-1] + (N,), dtype=x.dtype, device=x.device)
    o2 = out.view(-1, N)
    if rope is None:
        rc = _lib.load().dt_rmsnorm_qkv(_ptr(x2), x2.stride(0), _ptr(w_fused), _ptr(o2), o2.stride(0), M, K, N,
                                        float(eps), _dtype_code(x), _stream_ptr(x.device))
        _lib.check("dt_rmsnorm_qkv", rc)
        return out
    if x.dim() != 3:
        raise ValueError("rmsnorm_qkv with rope needs x of shape [B, S, K]")
    cos, sin = _prep_tables(rope[0], rope[1])
    rope_cols, head_dim = int(rope[2]), int(rope[3])
    rc = _lib.load().dt_rmsnorm_qkv_rope(_ptr(x2), x2.stride(0), _ptr(w_fused), _ptr(o2), o2.stride(0), M, K, N,
                                         float(eps), _ptr(cos), _ptr(sin), cos.stride(0), cos.shape[0], x.shape[1],
                                         rope_cols, head_dim, _dtype_code(x), _stream_ptr(x.device))
    _lib.check("dt_rmsnorm_qkv_rope", rc)
    return out


# ------------------------------------------------------------------ training operators
#
# A training step makes many small calls, and at small sizes the host's time for
# one (some 20 us) is the whole of it: these wrappers look at each tensor once
# and create no object that the call does not need.
def _same_device(first: Tensor, *ts: Optional[Tensor]) -> torch.device:
    """The device that every tensor is on (CUDA)."""
    dev = first.device
    if dev.type != "cuda":
        _require_cuda(first)
    for t in ts:
        if t is not None and t.device != dev:
            _require_cuda(t)
            raise ValueError(f"tensors are on different devices ({dev} and {t.device})")
    return dev


def _empty_as(t: Tensor) -> Tensor:
    """A contiguous tensor of t's shape and type (1.5 us on the host; from a shape and a type, 2.4 to 3.3)."""
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _launch(name: str, dev: torch.device, *args) -> None:
    """Calls the entry point on the device's current stream (its last argument), with the device
    current: the library launches there."""
    fn = getattr(_lib.load(), name)
    had = _raw_device() if _raw_device is not None else torch.cuda.current_device()
    if had == dev.index:
        rc = fn(*args, _stream_ptr(dev))
    else:
        torch.cuda.set_device(dev)
        try:
            rc = fn(*args, _stream_ptr(dev))
        finally:
            torch.cuda.set_device(had)
    if rc:
        _lib.check(name, rc)


@functools.lru_cache(maxsize=4096)
def _workspace(name: str, device: int, *sizes: int) -> int:
    """Bytes of scratch that the entry point ``name`` asks for (a rule on sizes and the device's SM count)."""
    with torch.cuda.device(device):
        size = getattr(_lib.load(), name)(*sizes)
    if size < 0:
        _lib.check(name, -size)
    return size


def _check_dropout(p: float, rng: Optional[Tensor], site: int) -> float:
    """The dropout arguments shared by the training operators; returns p as a float.

    ``rng``: int64 [2] device tensor (seed, step), see training.DropoutState;
    ``site``: a number of its own for each place of a model that drops."""
    p = float(p)
    if p != 0.0:
        if not 0.0 <= p < 1.0 or round(p * 65536) >= 65536:
            raise ValueError(f"dropout p must lie in [0, 1), below 1 - 2^-17 (got {p})")
        if rng is None:
            raise ValueError("dropout needs rng, an int64 [2] device tensor (seed, step)")
    if rng is not None and (rng.dtype != torch.int64 or rng.shape != (2,) or not rng.is_contiguous()):
        raise ValueError("rng must be a contiguous int64 tensor of shape [2] (seed, step)")
    if not 0 <= site < 2 ** 32:
        raise ValueError(f"site must lie in [0, 2^32) (got {site})")
    return p


def _rows16(t: Tensor) -> Tuple[Tensor, Tuple[int, int, int]]:
    """t when the attention kernels can read it ([B, S, H, D], contiguous D, strides multiples of 8,
    16-byte aligned), else a contiguous copy, and its first three strides."""
    b, s, h, d = t.stride()
    if d != 1 or (b | s | h) % 8 or b <= 0 or s <= 0 or h <= 0 or t.data_ptr() % 16:
        t = t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone()
        _, s, h, d = t.shape  # by its shape: the stride of a dimension of one element may be anything
        return t, (s * h * d, h * d, d)
    return t, (b, s, h)


def _check_attn_train(q: Tensor, k: Tensor, v: Tensor, pad_len: Optional[Tensor], scale: Optional[float]):
    if q.dim() != 4 or k.dim() != 4:
        raise ValueError("attn_train takes q [B, S, Hq, D] and k, v [B, S, Hkv, D]")
    B, S, Hq, D = q.shape
    kshape = k.shape
    if kshape != (B, S, kshape[2], D) or v.shape != kshape:
        raise ValueError(f"k/v shapes {tuple(k.shape)}, {tuple(v.shape)} do not match q {tuple(q.shape)}")
    if D not in (32, 64):
        raise ValueError(f"head_dim must be 32 or 64 (got {D})")
    dt = q.dtype
    if not (dt == k.dtype == v.dtype):
        raise TypeError("q, k, v must share a dtype")
    if dt not in (torch.bfloat16, torch.float16):
        raise TypeError(f"attn_train takes bf16 or fp16 (got {dt})")
    if pad_len is not None:
        if pad_len.shape != (B,):
            raise ValueError(f"pad_len must be [{B}] (got {tuple(pad_len.shape)})")
        if pad_len.dtype != torch.int32 or not pad_len.is_contiguous():
            pad_len = pad_len.to(torch.int32).contiguous()
    # As the kernels get it: a scale that fp32 holds as 0 would mean the default one.
    if scale is not None and not 0.0 < ctypes.c_float(scale).value < math.inf:
        raise ValueError(f"scale must be positive and finite in fp32 (got {scale})")
    if Hq < 1 or kshape[2] < 1 or Hq % kshape[2]:
        raise ValueError(f"{Hq} query heads are not a multiple of {kshape[2]} KV heads")
    return pad_len, B, S, Hq, kshape[2], D


def attn_train_forward(q: Tensor, k: Tensor, v: Tensor, pad_len: Optional[Tensor] = None,
                       scale: Optional[float] = None, p: float = 0.0, rng: Optional[Tensor] = None,
                       site: int = 0) -> Tuple[Tensor, Tensor]:
    """Causal GQA attention for training: q [B,S,Hq,D], k/v [B,S,Hkv,D] (rotated, bf16 / fp16) ->
    (out [B,S,Hq,D], lse [B,Hq,S] fp32, the backward call's input).

    pad_len [B] int32: leading padding positions.  Their rows of out are zeros and they pass no
    gradient (attn_prefill, the inference form, gives them the reference's mean of V).  p, rng,
    site: dropout on the attention weights, see _check_dropout."""
    dev = _same_device(q, k, v, pad_len, rng)
    pad_len, B, S, Hq, Hkv, D = _check_attn_train(q, k, v, pad_len, scale)
    p = _check_dropout(p, rng, site)
    (q, qs), (k, ks), (v, vs) = _rows16(q), _rows16(k), _rows16(v)
    out = _empty_as(q)
    lse = torch.empty(B, Hq, S, dtype=torch.float32, device=dev)
    if out.numel():
        size = _workspace("dt_attn_train_forward_workspace", dev.index, B, S, Hq, Hkv, D)
        ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
        _launch("dt_attn_train_forward", dev, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(),
                _ptr(pad_len), B, S, Hq, Hkv, D, *qs, *ks, *vs, S * Hq * D, Hq * D, D, _ptr(ws), size,
                scale or 0.0, p, _ptr(rng), site, _dtype_code(q))
    return out, lse


_PACK24 = struct.Struct("24q")


def attn_train_backward(dout: Tensor, q: Tensor, k: Tensor, v: Tensor, out: Tensor, lse: Tensor,
                        pad_len: Optional[Tensor] = None, scale: Optional[float] = None, p: float = 0.0,
                        rng: Optional[Tensor] = None, site: int = 0,
                        grads: Optional[Tuple[Tensor, Tensor, Tensor]] = None) -> Tuple[Tensor, Tensor, Tensor]:
    """Gradient of attn_train_forward: (dq, dk, dv) from dout and the forward call's arguments and
    results (the same rng contents, site and p).  ``grads``: tensors to write dq, dk and dv into
    (for instance the parts of one [B, S, Hq + 2 Hkv, D] gradient)."""
    dev = _same_device(q, k, v, dout, out, lse, pad_len, rng)
    pad_len, B, S, Hq, Hkv, D = _check_attn_train(q, k, v, pad_len, scale)
    p = _check_dropout(p, rng, site)
    dt = q.dtype
    if dout.shape != q.shape or out.shape != q.shape or dout.dtype != dt or out.dtype != dt:
        raise ValueError("dout and out must have q's shape and dtype")
    if lse.shape != (B, Hq, S) or lse.dtype != torch.float32 or not lse.is_contiguous():
        raise ValueError("lse must be the forward call's [B, Hq, S] fp32 tensor")
    (q, qs), (k, ks), (v, vs), (dout, dos), (out, os) = (_rows16(t) for t in (q, k, v, dout, out))
    if grads is None:
        dq, dk, dv = _empty_as(q), _empty_as(k), _empty_as(v)
        gs = (S * Hq * D, Hq * D, D) + 2 * (S * Hkv * D, Hkv * D, D)
    else:
        dq, dk, dv = grads
        _same_device(q, dq, dk, dv)
        gs = ()
        for name, t, like in (("dq", dq, q), ("dk", dk, k), ("dv", dv, v)):
            if t.shape != like.shape or t.dtype != dt or (t.numel() and _rows16(t)[0] is not t):
                raise ValueError(f"{name} must be a {tuple(like.shape)} {dt} tensor with contiguous D, 16-byte aligned "
                                 "rows and strides that are multiples of 8")
            gs += t.stride()[:3]
    if dq.numel():
        size = _workspace("dt_attn_train_workspace", dev.index, B, S, Hq, Hkv, D, int(p > 0.0))
        ws = torch.empty(size, dtype=torch.uint8, device=dev)
        _launch("dt_attn_train_backward", dev, dout.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                out.data_ptr(), lse.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _ptr(pad_len),
                ws.data_ptr(), size, B, S, Hq, Hkv, D, _PACK24.pack(*qs, *ks, *vs, *os, *dos, *gs), scale or 0.0, p,
                _ptr(rng), site, _dtype_code(q))
    return dq, dk, dv


def rope_grad_(g: Tensor, cos: Tensor, sin: Tensor, rope_cols: int, head_dim: int) -> Tensor:
    """Gradient of qkv_rope's rotation, in place: g [B, S, N] (the gradient of its output, contiguous)
    has its first rope_cols columns (the q and k heads) rotated back by table rows 0 .. S - 1."""
    dev = _same_device(g, cos, sin)
    if g.dim() != 3 or not g.is_contiguous():
        raise ValueError("rope_grad_ needs a contiguous [B, S, N] gradient")
    if not 0 < rope_cols <= g.shape[2]:
        raise ValueError(f"rope_cols {rope_cols} outside 1..{g.shape[2]}")
    if g.numel() == 0:
        return g
    cos, sin = _prep_tables(cos, sin)
    if cos.shape[-1] != head_dim or sin.shape != cos.shape:
        raise ValueError(f"cos / sin must be [rows, {head_dim}] tables")
    _launch("dt_rope_grad", dev, _ptr(g), g.stride(1), g.shape[0] * g.shape[1], _ptr(cos), _ptr(sin), cos.stride(0),
            cos.shape[0], g.shape[1], int(rope_cols), int(head_dim), _dtype_code(g))
    return g


def _check_width(n: int) -> None:
    """Widths go through the C ABI as 32-bit integers, which ctypes cuts without a word."""
    if n >= 2 ** 31:
        raise ValueError(f"rows of {n} elements are too wide: give them as more rows of fewer than 2^31 - 255")


def _rows2d(t: Tensor) -> Tuple[Tensor, int]:
    """t as [rows, K] with a contiguous last dimension (a copy when no view exists), and its row stride."""
    K = t.shape[-1]
    if t.is_contiguous():
        return t, K
    t2 = t.reshape(-1, K)
    if t2.stride(1) != 1 and K != 1:
        t2 = t2.contiguous()
    return t2, t2.stride(0)


def _gate_rows(gate: Tensor, x: Tensor) -> int:
    """The number of consecutive rows of x that share each row of the gate: a gate of shape [H], x's
    own shape, or x's shape with trailing ones before H ([B, 1, H] for [B, S, H])."""
    if gate.dim() > x.dim() or gate.dim() < 1 or gate.shape[-1] != x.shape[-1]:
        raise ValueError(f"gate {tuple(gate.shape)} does not broadcast to x {tuple(x.shape)}")
    lead = (1,) * (x.dim() - gate.dim()) + tuple(gate.shape[:-1])
    shared, shares = 1, False
    for g, n in zip(lead, x.shape[:-1]):
        if g == n and not (shares and n != 1):
            continue
        if g != 1:
            raise ValueError(f"gate {tuple(gate.shape)} must be x's shape {tuple(x.shape)} with ones in trailing places "
                             "before the last")
        shares = True
        shared *= n
    return shared


def _check_residual_norm(x, residual, pre_weight, post_weight, gate):
    dt, shape = x.dtype, x.shape
    if x.dim() < 1 or shape[-1] < 1:
        raise ValueError("x must have a last dimension")
    if dt not in _DTYPES:
        raise TypeError(f"unsupported dtype {dt}")
    _check_width(shape[-1])
    if residual is not None and residual.shape != shape:
        raise ValueError(f"residual {tuple(residual.shape)} does not match x {tuple(shape)}")
    if pre_weight.shape != shape[-1:] or not pre_weight.is_contiguous():
        raise ValueError(f"pre_weight must be a contiguous [{shape[-1]}] tensor")
    if post_weight is not None and (post_weight.shape != shape[-1:] or not post_weight.is_contiguous()):
        raise ValueError(f"post_weight must be a contiguous [{shape[-1]}] tensor")
    for t in (residual, pre_weight, post_weight, gate):
        if t is not None and t.dtype != dt:
            raise TypeError(f"residual, weights and gate must have x's dtype {dt} (got {t.dtype})")


def residual_norm_forward(x: Tensor, residual: Optional[Tensor], pre_weight: Tensor, eps: float,
                          post_weight: Optional[Tensor] = None, gate: Optional[Tensor] = None, alpha: float = 1.0,
                          p: float = 0.0, rng: Optional[Tensor] = None, site: int = 0) -> Tuple[Tensor, Tensor, Tensor]:
    """What stands between two products of a block, in one pass over x [..., H]:

        u = RMSNorm(x) * post_weight         (u = x without post_weight)
        h = residual + alpha * gate * dropout(u)
        n = RMSNorm(h) * pre_weight

    Returns (h, n, stats); stats [rows, 2] fp32 is the backward call's input.  ``gate``: [H], x's
    shape, or x's shape with ones in trailing places before H (a gate of each sample).  bf16, fp16
    or fp32, H <= 8192; fp32 arithmetic, each output rounded once, n from the unrounded h."""
    dev = _same_device(x, residual, pre_weight, post_weight, gate, rng)
    _check_residual_norm(x, residual, pre_weight, post_weight, gate)
    p = _check_dropout(p, rng, site)
    H = x.shape[-1]
    M = x.numel() // H
    x2, xs = _rows2d(x)
    r2, rs = (None, 0) if residual is None else _rows2d(residual)
    g2, gs, gate_rows = None, 0, 0
    if gate is not None:
        gate_rows = _gate_rows(gate, x)
        g2, gs = _rows2d(gate)
    h, n = _empty_as(x), _empty_as(x)
    stats = torch.empty(M, 2, dtype=torch.float32, device=dev)
    if M:
        _launch("dt_residual_norm_forward", dev, x2.data_ptr(), xs, _ptr(r2), rs, _ptr(g2), gs, gate_rows,
                pre_weight.data_ptr(), _ptr(post_weight), h.data_ptr(), n.data_ptr(), stats.data_ptr(), M, H, alpha,
                eps, p, _ptr(rng), site, _dtype_code(x))
    return h, n, stats


def residual_norm_backward(dh: Optional[Tensor], dn: Optional[Tensor], x: Tensor, residual: Optional[Tensor],
                           pre_weight: Tensor, stats: Tensor, post_weight: Optional[Tensor] = None,
                           gate: Optional[Tensor] = None, alpha: float = 1.0, p: float = 0.0,
                           rng: Optional[Tensor] = None, site: int = 0):
    """Gradient of residual_norm_forward from dh and dn (either may be None: zero):
    (dx, dresidual, dpre_weight, dpost_weight, dgate); the last two are None without their inputs.
    Sums over rows are fp32 and in a fixed order."""
    dev = _same_device(x, dh, dn, residual, pre_weight, post_weight, gate, stats, rng)
    _check_residual_norm(x, residual, pre_weight, post_weight, gate)
    p = _check_dropout(p, rng, site)
    shape, dt = x.shape, x.dtype
    for t in (dh, dn):
        if t is not None and (t.shape != shape or t.dtype != dt):
            raise ValueError("dh and dn must have x's shape and dtype")
    H = shape[-1]
    M = x.numel() // H
    if stats.shape != (M, 2) or stats.dtype != torch.float32 or not stats.is_contiguous():
        raise ValueError("stats must be the forward call's [rows, 2] fp32 tensor")
    gate_rows = 0 if gate is None else _gate_rows(gate, x)
    dx, dres = _empty_as(x), _empty_as(x)
    dpost = None if post_weight is None else _empty_as(post_weight)
    dgate = None if gate is None else _empty_as(gate)
    if M == 0 or (dh is None and dn is None):
        for t in (dx, dres, dpost, dgate):
            if t is not None:
                t.zero_()
        return dx, dres, torch.zeros_like(pre_weight), dpost, dgate
    dpre = torch.zeros_like(pre_weight) if dn is None else _empty_as(pre_weight)
    x2, xs = _rows2d(x)
    r2, rs = (None, 0) if residual is None else _rows2d(residual)
    g2, gs = (None, 0) if gate is None else _rows2d(gate)
    dh2, dhs = (None, 0) if dh is None else _rows2d(dh)
    dn2, dns = (None, 0) if dn is None else _rows2d(dn)
    size = _workspace("dt_residual_norm_workspace", dev.index, M, H, gate_rows, 0 if post_weight is None else 1)
    ws = torch.empty(size, dtype=torch.uint8, device=dev)
    _launch("dt_residual_norm_backward", dev, _ptr(dh2), dhs, _ptr(dn2), dns, x2.data_ptr(), xs, _ptr(r2), rs,
            _ptr(g2), gs, gate_rows, pre_weight.data_ptr(), _ptr(post_weight), stats.data_ptr(), dx.data_ptr(),
            dres.data_ptr(), dpre.data_ptr(), _ptr(dpost), _ptr(dgate), ws.data_ptr(), size, M, H, alpha, 0.0, p,
            _ptr(rng), site, _dtype_code(x))
    return dx, dres, dpre, dpost, dgate


def dropout_forward(x: Tensor, p: float, rng: Optional[Tensor], site: int = 0,
                    residual: Optional[Tensor] = None) -> Tensor:
    """residual + dropout(x) (residual None: dropout(x)) with a mask that is a function of rng, site
    and each element's place in x [..., H] and is never stored.  bf16, fp16 or fp32."""
    dev = _same_device(x, rng, residual)
    if x.dim() < 1 or x.dtype not in _DTYPES:
        raise TypeError(f"dropout takes bf16, fp16 or fp32 tensors of one or more dimensions (got {x.dtype})")
    _check_width(x.shape[-1])
    p = _check_dropout(p, rng, site)
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError("residual must have x's shape and dtype")
    y = _empty_as(x)
    n = y.numel()
    if n:
        H = x.shape[-1]
        x2, xs = _rows2d(x)
        r2, rs = (None, 0) if residual is None else _rows2d(residual)
        _launch("dt_dropout", dev, x2.data_ptr(), xs, _ptr(r2), rs, y.data_ptr(), H, n // H, H, p, _ptr(rng), site,
                _dtype_code(x))
    return y


def dropout_backward(dy: Tensor, p: float, rng: Optional[Tensor], site: int = 0) -> Tensor:
    """Gradient of dropout_forward with respect to x (its residual's gradient is dy itself)."""
    return dropout_forward(dy, p, rng, site)

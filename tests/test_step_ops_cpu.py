"""Refusals of the head norms that need no GPU."""
import pytest
import torch


def test_head_norm_entry_points_refuse_bad_arguments():
    from rl_for_mario_b200 import _lib

    lib = _lib.load()
    a, INV, UNS = 4096, _lib.DT_ERR_INVALID, _lib.DT_ERR_UNSUPPORTED

    def fwd(q=a, out=a, cos=a, cos_stride=32, rows=8, start=None, B=1, S=8, Hq=4, Hkv=2, D=32, strides=(8,) * 12,
            w=a, w32=0, eps=1e-5, dtype=0):
        st = (_lib._L * len(strides))(*strides) if strides else None
        return lib.dt_head_norm_rope_forward(q, a, w, a, out, a, cos, a, cos_stride, rows, start, B, S, Hq, Hkv, D, st,
                                             w32, eps, dtype, None)

    for kw, code in ((dict(q=None), INV), (dict(out=None), INV), (dict(w=None), INV), (dict(cos=None), INV),
                     (dict(strides=None), INV), (dict(B=0), INV), (dict(S=0), INV), (dict(Hkv=0), INV),
                     (dict(D=33), UNS), (dict(D=0), UNS), (dict(D=258), UNS), (dict(dtype=3), UNS),
                     (dict(q=a + 1), INV), (dict(w=a + 2, w32=1), INV), (dict(cos=a + 2), INV),
                     (dict(start=a + 2), INV), (dict(rows=7), INV), (dict(rows=0, start=a), INV),
                     (dict(cos_stride=31), INV), (dict(strides=(-8,) + (8,) * 11), INV), (dict(eps=-1.0), INV),
                     (dict(eps=float("nan")), INV), (dict(B=1 << 20, S=1 << 10, start=a), UNS)):
        assert fwd(**kw) == code, kw

    def bwd(g=a, dw=a, ws=a, size=1 << 30):
        st = (_lib._L * 18)(*(8,) * 18)
        return lib.dt_head_norm_rope_backward(g, a, a, a, a, a, a, a, dw, a, a, a, 32, 8, None, ws, size, 1, 8, 4, 2, 32,
                                              st, 0, 1e-5, 0, None)

    assert bwd(g=None) == INV and bwd(dw=None) == INV
    assert lib.dt_head_norm_rope_workspace(1, 8, 4, 2, 31) < 0 and lib.dt_head_norm_rope_workspace(0, 8, 4, 2, 32) < 0


def test_head_norm_wrapper_checks():
    from rl_for_mario_b200 import kernels as K

    q, k, w = torch.zeros(2, 4, 4, 32), torch.zeros(2, 4, 2, 32), torch.ones(32)
    t = torch.zeros(4, 32)
    with pytest.raises(ValueError, match="CUDA"):
        K.head_norm_rope_forward(q, k, w, w, 1e-5, t, t)
    with pytest.raises(ValueError, match="CUDA"):
        K.head_norm_rope_backward(q, k, q, k, w, w, 1e-5, t, t)
    ok = (q, k, w, w, 1e-5, t, t, None)
    assert K._check_head_norm(*ok)[3:] == (2, 4, 4, 2, 32)

    def refused(kind, match, **kw):
        names = ("q", "k", "q_weight", "k_weight", "eps", "cos", "sin", "start_pos")
        args = dict(zip(names, ok))
        args.update(kw)
        with pytest.raises(kind, match=match):
            K._check_head_norm(**args)

    refused(ValueError, "takes q", q=q[0])
    refused(ValueError, "match", k=k[:1])
    refused(TypeError, "dtype", k=k.half())
    refused(TypeError, "dtype", q=q.double(), k=k.double())
    refused(ValueError, "even", q=torch.zeros(2, 4, 4, 31), k=torch.zeros(2, 4, 2, 31))
    refused(ValueError, "even", q=torch.zeros(2, 4, 1, 258), k=torch.zeros(2, 4, 1, 258))
    refused(ValueError, "one head", k=k[:, :, :0])
    refused(ValueError, "2.31", q=torch.empty(2, 4, 4, 32).expand(2, 4, 4, 32).as_strided((2 ** 16, 2 ** 15, 4, 32), (0, 0, 0, 1)),
            k=torch.empty(32).as_strided((2 ** 16, 2 ** 15, 2, 32), (0, 0, 0, 1)))
    refused(ValueError, "contiguous", q_weight=torch.ones(64)[::2])
    refused(ValueError, "contiguous", k_weight=torch.ones(31))
    refused(TypeError, "fp32", q_weight=w.half())
    refused(TypeError, "fp32", q_weight=w.half(), k_weight=w.half())
    refused(ValueError, "eps", eps=-1.0)
    refused(ValueError, "eps", eps=float("nan"))
    refused(ValueError, "eps", eps=1e39)
    refused(ValueError, "tables", cos=t[:3], sin=t[:3])
    refused(ValueError, "tables", cos=t[:, :16], sin=t[:, :16])
    refused(ValueError, "tables", sin=torch.zeros(5, 32))
    refused(ValueError, "start_pos", start_pos=torch.zeros(3, dtype=torch.int32))
    assert K._check_head_norm(*ok[:7], torch.zeros(2, dtype=torch.int64))[2].dtype == torch.int32

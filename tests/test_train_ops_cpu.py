"""Refusals of the training operators that need no GPU: entry points and wrappers check their
arguments before any device work.  And the generator's published properties on the CPU."""
import numpy as np
import pytest
import torch

from oracle import train_ref as ref


def test_entry_points_refuse_bad_arguments_without_a_gpu():
    from rl_for_mario_b200 import _lib

    lib = _lib.load()
    s12, a = [256, 64, 64] * 4, 4096  # any aligned non-null address: nothing is read before the device check

    def fwd(q=a, S=8, Hq=4, Hkv=2, D=32, strides=s12, p=0.0, rng=None, dtype=0, B=1):
        return lib.dt_attn_train_forward(q, a, a, a, a, None, B, S, Hq, Hkv, D, *strides, None, 0, 0.0, p, rng, 0, dtype, None)

    cases = [(dict(q=None), "null", _lib.DT_ERR_INVALID), (dict(S=0), "positive", _lib.DT_ERR_INVALID),
             (dict(Hkv=3), "divisible", _lib.DT_ERR_INVALID), (dict(D=48), "head_dim", _lib.DT_ERR_UNSUPPORTED),
             (dict(dtype=2), "dtype", _lib.DT_ERR_UNSUPPORTED), (dict(q=a + 2), "aligned", _lib.DT_ERR_INVALID),
             (dict(strides=[257] + s12[1:]), "multiple of 8", _lib.DT_ERR_INVALID),
             (dict(strides=[0] + s12[1:]), "multiple of 8", _lib.DT_ERR_INVALID),
             (dict(p=1.0), "p must lie", _lib.DT_ERR_INVALID), (dict(p=-0.1), "p must lie", _lib.DT_ERR_INVALID),
             (dict(p=float("nan")), "p must lie", _lib.DT_ERR_INVALID),
             (dict(p=0.999995), "rounds to 1", _lib.DT_ERR_INVALID), (dict(p=0.1), "null rng", _lib.DT_ERR_INVALID),
             (dict(p=0.1, rng=a + 4), "8-byte", _lib.DT_ERR_INVALID),
             (dict(B=1 << 30, S=1 << 20), "too many", _lib.DT_ERR_UNSUPPORTED)]
    for kw, text, code in cases:
        assert fwd(**kw) == code and text.encode() in lib.dt_last_error(), kw
    s24 = (_lib._L * 24)(*([256, 64, 64] * 8))

    def bwd(dq=a, ws=a, dtype=0):
        return lib.dt_attn_train_backward(a, a, a, a, a, a, dq, a, a, None, ws, 1 << 20, 1, 8, 4, 2, 32, s24, 0.0, 0.0,
                                          None, 0, dtype, None)

    assert bwd(ws=None) == _lib.DT_ERR_INVALID and bwd(dq=a + 8) == _lib.DT_ERR_INVALID
    assert bwd(dtype=2) == _lib.DT_ERR_UNSUPPORTED
    assert lib.dt_attn_train_workspace(1, 8, 4, 3, 32, 0) < 0 and lib.dt_attn_train_workspace(1, 0, 4, 2, 32, 1) < 0

    def norm(x=a, w=a, gate=None, gate_rows=0, M=4, H=8, dtype=0, h=a, p=0.0):
        return lib.dt_residual_norm_forward(x, 8, a, 8, gate, 8, gate_rows, w, None, h, a, a, M, H, 1.0, 1e-5, p, None,
                                            0, dtype, None)

    for kw in (dict(x=None), dict(w=None), dict(h=None), dict(M=0), dict(H=0), dict(gate=a, gate_rows=3),
               dict(gate=a, gate_rows=0), dict(x=a + 1), dict(p=0.1), dict(dtype=1, x=a + 1)):
        assert norm(**kw) == _lib.DT_ERR_INVALID, kw
    assert norm(H=8193) == _lib.DT_ERR_UNSUPPORTED and norm(dtype=5) == _lib.DT_ERR_UNSUPPORTED
    assert lib.dt_residual_norm_workspace(4, 8193, 0, 0) < 0 and lib.dt_residual_norm_workspace(4, 8, 3, 0) < 0
    assert lib.dt_residual_norm_backward(None, 8, None, 8, a, 8, a, 8, None, 0, 0, a, None, a, a, a, a, None, None, a,
                                         1 << 20, 4, 8, 1.0, 0.0, 0.0, None, 0, 0, None) == _lib.DT_ERR_INVALID
    for kw in (dict(x=None), dict(y=None), dict(rows=0), dict(cols=0), dict(x=a + 1)):
        d = dict(x=a, y=a, rows=4, cols=8, **{})
        d.update(kw)
        assert lib.dt_dropout(d["x"], 8, None, 0, d["y"], 8, d["rows"], d["cols"], 0.0, None, 0, 0,
                              None) == _lib.DT_ERR_INVALID, kw


def test_wrappers_refuse_cpu_tensors():
    from rl_for_mario_b200 import kernels

    q, k = torch.zeros(1, 4, 4, 32, dtype=torch.bfloat16), torch.zeros(1, 4, 2, 32, dtype=torch.bfloat16)
    x, w = torch.zeros(2, 8), torch.ones(8)
    with pytest.raises(ValueError, match="CUDA"):
        kernels.attn_train_forward(q, k, k)
    with pytest.raises(ValueError, match="CUDA"):
        kernels.attn_train_backward(q, q, k, k, q, torch.zeros(1, 4, 4))
    with pytest.raises(ValueError, match="CUDA"):
        kernels.residual_norm_forward(x, x, w, 1e-5)
    with pytest.raises(ValueError, match="CUDA"):
        kernels.residual_norm_backward(x, x, x, x, w, torch.zeros(2, 2))
    with pytest.raises(ValueError, match="CUDA"):
        kernels.dropout_forward(x, 0.1, torch.zeros(2, dtype=torch.int64))


def test_argument_checks_on_the_host():
    from rl_for_mario_b200 import kernels as K

    x = torch.zeros(2, 3, 8)
    for shape, shared in (((8,), 6), ((1, 8), 6), ((2, 1, 8), 3), ((1, 1, 8), 6), ((2, 3, 8), 1)):
        assert K._gate_rows(torch.zeros(shape), x) == shared
    for shape in ((3, 8), (1, 3, 8), (7,), (1, 2, 3, 8), (2, 2, 8)):
        with pytest.raises(ValueError, match="gate"):
            K._gate_rows(torch.zeros(shape), x)
    one = torch.zeros(1, 3, 8)
    assert K._gate_rows(torch.zeros(1, 1, 8), one) == 3 and K._gate_rows(torch.zeros(3, 8), one) == 1
    with pytest.raises(TypeError, match="dtype"):
        K._check_residual_norm(x, x.bfloat16(), torch.ones(8), None, None)
    with pytest.raises(ValueError, match="residual"):
        K._check_residual_norm(x, x[:1], torch.ones(8), None, None)
    with pytest.raises(ValueError, match="pre_weight"):
        K._check_residual_norm(x, None, torch.ones(7), None, None)
    rng = torch.zeros(2, dtype=torch.int64)
    assert K._check_dropout(0, None, 0) == 0.0 and K._check_dropout(0.5, rng, 2 ** 32 - 1) == 0.5
    for p, r, site in ((1.0, rng, 0), (-0.1, rng, 0), (float("nan"), rng, 0), (0.1, None, 0), (0.1, rng.int(), 0),
                       (0.1, rng[:1], 0), (0.1, rng, -1), (0.1, rng, 2 ** 32), (0.999995, rng, 0)):
        with pytest.raises(ValueError):
            K._check_dropout(p, r, site)
    q, k = torch.zeros(1, 4, 4, 32, dtype=torch.bfloat16), torch.zeros(1, 4, 2, 32, dtype=torch.bfloat16)
    with pytest.raises(TypeError, match="bf16"):
        K._check_attn_train(q.float(), k.float(), k.float(), None, None)
    with pytest.raises(ValueError, match="pad_len"):
        K._check_attn_train(q, k, k, torch.zeros(2), None)
    with pytest.raises(ValueError, match="scale"):
        K._check_attn_train(q, k, k, None, 0.0)
    with pytest.raises(ValueError, match="shapes"):
        K._check_attn_train(q, k, k[:, :3], None, None)


def test_generator_words():
    """Every word takes each half equally often, blocks differ in every counter and key word, and the
    64-bit multiplication agrees with Python's integers."""
    w = ref.philox_words(np.arange(1 << 14, dtype=np.uint64), 12345, 6, 7)
    # 2^14 draws a word: six standard deviations of a fair bit.
    assert (np.abs((w >= 32768).mean(0) - 0.5) <= 6 * 0.5 / 128).all()
    base = ref.philox_words(np.array([5], dtype=np.uint64), 1, 2, 3)
    for args in ((6, 1, 2, 3), (5 + (1 << 32), 1, 2, 3), (5, 2, 2, 3), (5, 1 + (1 << 32), 2, 3), (5, 1, 3, 3),
                 (5, 1, 2, 4)):
        assert not np.array_equal(base, ref.philox_words(np.array([args[0]], dtype=np.uint64), *args[1:]))
    c, k = [5, 0, 2, 3], [1, 0]
    for _ in range(7):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    assert base[0].tolist() == [h for v in c for h in (v & 0xFFFF, v >> 16)]


def test_streams_and_devices_of_a_launch(monkeypatch):
    """The stream of a device named with and without an index, with and without torch's private shortcuts; a launch
    makes its tensors' device current and puts the other one back, also when the call raises."""
    from types import SimpleNamespace

    from rl_for_mario_b200 import kernels as K

    monkeypatch.setattr(torch.cuda, "current_stream", lambda d: SimpleNamespace(cuda_stream=100 + (d.index or 0)))
    monkeypatch.setattr(K, "_raw_stream", lambda i: 100 + i)
    one, bare = torch.device("cuda", 1), torch.device("cuda")
    assert K._stream_ptr(one) == 101 and K._stream_ptr(bare) == 100
    monkeypatch.setattr(K, "_raw_stream", None)
    assert K._stream_ptr(one) == 101 and K._stream_ptr(bare) == 100

    now, seen = [0], []

    def entry(*args):
        seen.append((now[0], args))
        if args[0] == "raise":
            raise RuntimeError("from the call")
        return 0

    monkeypatch.setattr(K._lib, "load", lambda: SimpleNamespace(entry=entry))
    monkeypatch.setattr(torch.cuda, "set_device", lambda d: now.__setitem__(0, d if isinstance(d, int) else d.index))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: now[0])
    for raw in (lambda: now[0], None):
        monkeypatch.setattr(K, "_raw_device", raw)
        K._launch("entry", one, "a")
        assert seen[-1] == (1, ("a", 101)) and now[0] == 0
        with pytest.raises(RuntimeError, match="from the call"):
            K._launch("entry", one, "raise")
        assert now[0] == 0
        K._launch("entry", torch.device("cuda", 0), "b")
        assert seen[-1] == (0, ("b", 100)) and now[0] == 0


def test_widths_beyond_32_bits_are_refused(monkeypatch):
    """2^32 + 8 columns would reach the library as 8; from 2^31 - 255 on the kernel's column numbers would overflow."""
    from rl_for_mario_b200 import _lib, kernels as K

    lib, a = _lib.load(), 4096
    for cols in (2 ** 31 - 255, 2 ** 31 - 1):
        assert lib.dt_dropout(a, 8, None, 0, a, 8, 1, cols, 0.0, None, 0, 0, None) == _lib.DT_ERR_UNSUPPORTED
    rows = torch.empty(1, device="meta", dtype=torch.bfloat16)
    for n in (2 ** 31, 2 ** 32 + 8):
        wide = rows.expand(2, n)
        with pytest.raises(ValueError, match="too wide"):
            K._check_residual_norm(wide, None, wide[0], None, None)
        monkeypatch.setattr(K, "_same_device", lambda *t: torch.device("cuda", 0))
        with pytest.raises(ValueError, match="too wide"):
            K.dropout_forward(wide, 0.0, None)


def heads(h):
    return torch.zeros(1, 4, h, 32, dtype=torch.bfloat16)


def test_scales_that_fp32_does_not_hold():
    """A scale that fp32 rounds to 0 stood for the default one."""
    from rl_for_mario_b200 import kernels as K

    for scale in (1e-50, -1.0, float("nan"), float("inf"), 1e39):
        with pytest.raises(ValueError, match="scale"):
            K._check_attn_train(heads(4), heads(2), heads(2), None, scale)
    assert K._check_attn_train(heads(4), heads(2), heads(2), None, 1e-30)[1:] == (1, 4, 4, 2, 32)


def test_numbers_of_heads():
    """No query heads left dk and dv unwritten, whatever the number of KV heads."""
    from rl_for_mario_b200 import kernels as K

    for hq, hkv in ((0, 2), (4, 0), (0, 0), (3, 2), (2, 4)):
        with pytest.raises(ValueError, match="heads"):
            K._check_attn_train(heads(hq), heads(hkv), heads(hkv), None, None)

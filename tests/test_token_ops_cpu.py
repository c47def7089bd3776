"""Refusals of the token operators (layer norm, dropout, rotary positions): every bad argument is turned down on the host, before
anything is launched -- by the Python layer and by the C entry points themselves."""
import ctypes

import pytest
import torch

from indm_amd import hip, ops

F32, BF16 = torch.float32, torch.bfloat16


def t(*shape, dtype=F32):
    return torch.zeros(shape, dtype=dtype)


@pytest.mark.parametrize("args,what", [
    ((t(4, 8, dtype=torch.float16),), "float32 or bfloat16"),
    ((t(4, 8), t(7)), r"gamma is \[8\]"),
    ((t(4, 8), t(8, dtype=BF16)), "gamma is float32"),
    ((t(4, 8), t(8), t(1, 8)), r"beta is \[8\]"),
    ((t(4, 0),), "not empty"),
    ((t(1, 16385),), "16384"),
    ((t(1, 16385, dtype=BF16),), "16384"),
    ((t(4, 8), None, None, -1e-6), "eps >= 0"),
    ((t(4, 8),), "no CPU fallback"),
])
def test_layer_norm_refuses(args, what):
    with pytest.raises(RuntimeError, match=what):
        ops.layer_norm(*args)


@pytest.mark.parametrize("args,kw,what", [
    ((t(8, dtype=torch.float64), 0.1, 1), {}, "float32 or bfloat16"),
    ((t(8), -0.1, 1), {}, "0 <= p <= 1"),
    ((t(8), 1.5, 1), {}, "0 <= p <= 1"),
    ((t(8), float("nan"), 1), {}, "0 <= p <= 1"),
    ((t(8), 0.1, -1), {}, "seed"),
    ((t(8), 0.1, 1 << 64), {}, "seed"),
    ((t(8), 0.1, 1), dict(res=t(1, 8)), "res is"),
    ((t(8), 0.1, 1), dict(res=t(8, dtype=BF16)), "res is"),
    ((t(8), 0.1, 1), {}, "no CPU fallback"),
])
def test_dropout_refuses(args, kw, what):
    with pytest.raises(RuntimeError, match=what):
        ops.dropout(*args, **kw)


def _rot(q=None, k=None, pos=None, freqs=None, sections=(4, 4), **kw):
    q = t(2, 5, 3, 16) if q is None else q
    pos = t(5, 2, dtype=torch.int32) if pos is None else pos
    freqs = ops.rotary_freqs((4, 4)) if freqs is None else freqs
    return ops.rotary(q, k, pos, freqs, sections, **kw)


@pytest.mark.parametrize("kw,what", [
    (dict(q=t(5, 3, 16)), r"q is \[B, T, H, D\]"),
    (dict(q=t(2, 5, 3, 16, dtype=torch.float16)), "float32 or bfloat16"),
    (dict(k=t(2, 5, 3, 8)), "k is"),
    (dict(k=t(2, 4, 3, 16)), "k is"),
    (dict(k=t(2, 5, 3, 16, dtype=BF16)), "k is"),
    (dict(sections=(3, 5)), "even positive"),
    (dict(sections=()), "even positive"),
    (dict(sections=(16, 2)), "even positive"),
    (dict(sections=(-2, 10)), "even positive"),
    (dict(sections=(2,) * 9, q=t(2, 5, 3, 32)), "even positive"),
    (dict(q=t(1, 5, 1, 4098)), "up to 4096"),
    (dict(pos=t(5, 3, dtype=torch.int32)), "pos is"),
    (dict(pos=t(1, 5, 2, dtype=torch.int32)), "pos is"),
    (dict(pos=t(5, 2, dtype=torch.float64)), "positions are"),
    (dict(freqs=ops.rotary_freqs((4, 6))), "freqs is"),
    (dict(freqs=ops.rotary_freqs((4, 4)).float()), "freqs is"),
    (dict(freqs=ops.rotary_freqs((4, 4)).requires_grad_()), "no gradient"),
    (dict(pos=t(5, 2).requires_grad_()), "no gradient"),
    ({}, "no CPU fallback"),
])
def test_rotary_refuses(kw, what):
    with pytest.raises(RuntimeError, match=what):
        _rot(**kw)


def test_rotary_freqs():
    f = ops.rotary_freqs((4, 6), base=100.0)
    want = torch.tensor([1.0, 100.0 ** -0.5, 1.0, 100.0 ** (-1 / 3), 100.0 ** (-2 / 3)], dtype=torch.float64)
    assert f.dtype == torch.float64 and torch.allclose(f, want, rtol=1e-15)


def test_c_entry_points_refuse_and_ignore_empty_work():
    """the C ABI by itself: bad sizes and null pointers come back as a status, empty problems as success, nothing is launched"""
    L, buf = hip.lib(), (ctypes.c_float * 64)()
    p = ctypes.addressof(buf)
    for suf, most in (("f32", 16384), ("bf16", 16384)):
        fwd, bwd = getattr(L, "indm_layernorm_fwd_" + suf), getattr(L, "indm_layernorm_bwd_" + suf)
        assert fwd(p, 8, None, None, p, None, None, 4, 0, 1e-6, None) == -1
        assert fwd(p, 8, None, None, p, None, None, 4, most + 1, 1e-6, None) == -1
        assert fwd(p, 8, None, None, p, None, None, -1, 8, 1e-6, None) == -1
        assert fwd(p, 8, None, None, p, p, None, 4, 8, 1e-6, None) == -4
        assert fwd(None, 8, None, None, p, None, None, 4, 8, 1e-6, None) == -4
        assert fwd(None, 8, None, None, None, None, None, 0, 8, 1e-6, None) == 0
        assert bwd(p, p, 8, None, p, p, p, p, p, None, 4, 8, None) == -4          # the parameters' gradients need the scratch
        assert bwd(p, p, 8, None, None, p, p, None, None, None, 4, 8, None) == -4
        assert bwd(p, p, 8, None, p, p, p, None, None, None, 4, most + 1, None) == -1
        assert bwd(None, None, 8, None, None, None, None, None, None, None, 0, 8, None) == 0
        drop = getattr(L, "indm_dropout_" + suf)
        assert drop(p, None, p, -1, 0.1, 1, None, None) == -1
        assert drop(p, None, p, 8, 1.1, 1, None, None) == -4
        assert drop(p, None, p, 8, float("nan"), 1, None, None) == -4
        assert drop(None, None, p, 8, 0.1, 1, None, None) == -4
        assert drop(None, None, None, 0, 0.1, 1, None, None) == 0
        rot = getattr(L, "indm_rotary_" + suf)
        st, sec = (ctypes.c_long * 6)(), (ctypes.c_int * 2)(4, 4)
        assert rot(p, None, p, None, st, 1, 1, 1, 0, 6, p, 0, 0, p, sec, 2, 0, 0, None) == -1     # sections past the head
        assert rot(p, None, p, None, st, 1, 1, 1, 0, 16, p, 0, 0, p, (ctypes.c_int * 2)(3, 4), 2, 0, 0, None) == -1
        assert rot(p, None, p, None, st, 1, 1, 1, 0, 16, p, 0, 0, p, sec, 9, 0, 0, None) == -1
        assert rot(p, None, p, None, st, 1, 1, 1, 0, 16, p, 3, 0, p, sec, 2, 0, 0, None) == -4
        assert rot(p, None, p, None, st, 2, 3, 1, 0, 16, p, 0, 5, p, sec, 2, 0, 0, None) == -4     # (samples' positions lie one after the other)
        assert rot(p, None, p, None, None, 1, 1, 1, 0, 16, p, 0, 0, p, sec, 2, 0, 0, None) == -4
        assert rot(None, None, p, None, st, 1, 1, 1, 0, 16, p, 0, 0, p, sec, 2, 0, 0, None) == -4
        assert rot(p, None, p, None, st, 1, 1, 1, 1, 16, p, 0, 0, p, sec, 2, 0, 0, None) == -4
        assert rot(None, None, None, None, st, 0, 1, 1, 0, 16, None, 0, 0, None, sec, 2, 0, 0, None) == 0
    assert L.indm_layernorm_bwd_ws_floats(0, 8, 4) == 0 and L.indm_layernorm_bwd_ws_floats(8, 8, 3) == 0
    assert L.indm_layernorm_bwd_ws_floats(1, 8, 2) == 16

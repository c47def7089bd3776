"""Refusals of window attention: bad arguments are turned down on the host, by the Python layer and by the C entry points."""
import ctypes

import pytest
import torch

from indm_amd import hip, ops


def t(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


def call(q=None, k=None, v=None, **kw):
    q = t(2, 5, 4, 16) if q is None else q
    k = t(2, 5, 2, 16) if k is None else k
    return ops.window_attention(q, k, t(*k.shape, dtype=k.dtype) if v is None else v, **kw)


@pytest.mark.parametrize("kw,what", [
    (dict(q=t(2, 5, 4, 16, dtype=torch.float16)), "float32 or bfloat16"),
    (dict(q=t(5, 4, 16)), r"q is \[B, T, H, D\]"),
    (dict(q=t()), r"q is \[B, T, H, D\]"),
    (dict(q=t(2, 5, 4, 0), k=t(2, 5, 4, 0)), "8, 16"),
    (dict(k=t(2, 4, 2, 16)), "k is"),
    (dict(k=t(2, 5, 2, 8)), "k is"),
    (dict(k=t(2, 5, 2, 16, dtype=torch.bfloat16)), "k is"),
    (dict(v=t(2, 5, 4, 16)), "v is"),
    (dict(v=t(2, 5, 2, 16, dtype=torch.bfloat16)), "v is"),
    (dict(k=t(2, 5, 3, 16)), "multiple of the 3"),
    (dict(k=t(2, 5, 0, 16)), "multiple of the 0"),
    (dict(q=t(2, 5, 4, 12), k=t(2, 5, 4, 12)), "8, 16"),
    (dict(q=t(2, 5, 4, 136), k=t(2, 5, 4, 136)), "8, 16"),
    (dict(window=-1), "window and sinks"),
    (dict(window=(3, -2)), "window and sinks"),
    (dict(sinks=-1), "window and sinks"),
    (dict(scale=0.0), "scale > 0"),
    (dict(scale=-1.0), "scale > 0"),
    (dict(scale=float("nan")), "scale > 0"),
    (dict(scale=float("inf")), "scale > 0"),
    (dict(lengths=torch.zeros(2, dtype=torch.int64)), "lengths is int32"),
    (dict(lengths=torch.zeros(3, dtype=torch.int32)), "lengths is int32"),
    ({}, "no CPU fallback"),
])
def test_window_attention_refuses(kw, what):
    with pytest.raises(RuntimeError, match=what):
        call(**kw)


def test_c_entry_points_refuse_and_ignore_empty_work():
    L = hip.lib()
    buf = (ctypes.c_char * 512)()
    p = (ctypes.addressof(buf) + 63) // 64 * 64
    for suf in ("f32", "bf16"):
        fwd, bwd = getattr(L, "indm_wattn_fwd_" + suf), getattr(L, "indm_wattn_bwd_" + suf)
        ok = (ctypes.c_long * 9)(*[64] * 9)

        def f(q=p, s=ok, o=p, B=1, T=4, H=2, Hk=1, D=16, l=1, r=1, sinks=0, scale=1.0):
            return fwd(q, p, p, s, o, None, None, None, B, T, H, Hk, D, l, r, sinks, 0, scale, None)

        def g(ws=p, o=p, D=16, T=4):
            return bwd(p, p, p, ok, o, None, p, p, None, p, p, p, ws, 1, T, 2, 1, D, 1, 1, 0, 0, 1.0, None)

        assert f(H=3, Hk=2) == f(D=12) == f(D=136) == f(D=0) == f(B=-1) == f(T=-1) == f(T=(1 << 28) + 1) == f(H=0) == f(Hk=0) == -1
        assert f(l=-1) == f(r=-1) == f(sinks=-1) == f(scale=0.0) == f(scale=float("nan")) == f(scale=float("inf")) == -4
        assert f(s=None) == f(q=None) == f(q=p + 8) == f(o=None) == f(o=p + 4) == -4
        assert f(s=(ctypes.c_long * 9)(*[64] * 8, 3)) == f(s=(ctypes.c_long * 9)(-64, *[64] * 8)) == -4
        assert f(s=(ctypes.c_long * 9)(64, 1 << 23, *[64] * 7)) == f(H=1 << 20, Hk=1) == -1
        assert f(B=0, q=None) == f(T=0, q=None) == 0
        assert g(ws=None) == g(ws=p + 4) == g(o=None) == g(o=p + 8) == -4
        assert g(D=20) == -1 and g(T=0) == 0
    ws = L.indm_wattn_bwd_ws_floats
    assert ws(1, 0, 2, 1, 16, 1, 1, 0, 0) == 0 and ws(1, 4, 3, 2, 16, 1, 1, 0, 0) == 0
    assert ws(2, 5, 4, 2, 16, 1, 1, 0, 0) == 40                  # <dO, o> of every query
    assert ws(2, 5, 4, 2, 16, 5, 5, 3, 0) == 40                  # windows that see everything: the sinks add nothing
    assert ws(1, 64, 1, 1, 16, 5, 5, 3, 0) == 64 + 2 * 3 * 2 * 16    # the three sinks' dk, dv: one share from all queries, one from the window

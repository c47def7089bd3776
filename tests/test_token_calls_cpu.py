"""Ways of calling the token operators that they refuse rather than answer wrongly, whatever device the tensors are on."""
import ctypes

import pytest
import torch
from torch.autograd import forward_ad

from indm_amd import hip, ops

X, G, POS, FREQS = torch.ones(2, 3, 2, 8), torch.ones(8), torch.zeros(3, 1), ops.rotary_freqs((8,))
CALLS = {
    "layer_norm": (lambda x: ops.layer_norm(x), X),
    "layer_norm gamma": (lambda g: ops.layer_norm(X, g), G),
    "layer_norm beta": (lambda b: ops.layer_norm(X, None, b), G),
    "dropout": (lambda x: ops.dropout(x, 0.5, 1), X),
    "dropout res": (lambda r: ops.dropout(X, 0.5, 1, res=r), X),
    "rotary": (lambda q: ops.rotary(q, None, POS, FREQS, (8,))[0], X),
    "rotary k": (lambda k: ops.rotary(X, k, POS, FREQS, (8,))[1], X),
    "rotary pos": (lambda p: ops.rotary(X, None, p, FREQS, (8,))[0], POS),
    "rotary freqs": (lambda f: ops.rotary(X, None, POS, f, (8,))[0], FREQS),
    "window_attention q": (lambda q: ops.window_attention(q, X, X, 1), X),
    "window_attention k": (lambda k: ops.window_attention(X, k, X, 1), X),
    "window_attention v": (lambda v: ops.window_attention(X, X, v, 1), X),
}


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused(name, grad):
    """a dual tensor does not require grad: its tangent would be lost without a word"""
    call, x = CALLS[name]
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        with pytest.raises(RuntimeError, match="forward-mode"):
            call(forward_ad.make_dual(x, torch.ones_like(x)))


@pytest.mark.parametrize("name", ["layer_norm", "dropout", "rotary", "window_attention q"])
def test_tracing_is_refused(name):
    call, x = CALLS[name]
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(call, (x.clone(),), check_trace=False)


@pytest.mark.parametrize("which", ["q heads", "k heads", "samples"])
def test_rotary_refuses_what_does_not_fit_32_bits(which):
    """counts that the kernel holds in 32 bits: a number past them would be taken for a small one"""
    many = (1 << 32) + 1
    q = torch.ones(1, 1, 1, 8).expand(many if which == "samples" else 1, 1, many if which == "q heads" else 1, 8)
    k = torch.ones(1, 1, 1, 8).expand(1, 1, many, 8) if which == "k heads" else None
    with pytest.raises(RuntimeError, match="samples and heads"):
        ops.rotary(q, k, torch.zeros(1, 1), FREQS, (8,))


def test_gradients_that_are_not_wanted():
    """the C entry points: no gradient wanted is no work, dk and dv come together"""
    buf = (ctypes.c_char * 512)()
    p = (ctypes.addressof(buf) + 63) // 64 * 64
    strides = (ctypes.c_long * 9)(*[64] * 9)
    for suf in ("f32", "bf16"):
        norm, attn = getattr(hip.lib(), "indm_layernorm_bwd_" + suf), getattr(hip.lib(), "indm_wattn_bwd_" + suf)
        assert norm(p, p, 8, None, p, p, None, None, None, None, 4, 8, None) == 0
        assert norm(p, p, 8, None, p, p, None, p, None, None, 4, 8, None) == -4      # (the parameters' gradients need the scratch)

        def f(dq, dk, dv):
            return attn(p, p, p, strides, p, None, p, p, None, dq, dk, dv, p, 1, 4, 2, 1, 16, 1, 1, 0, 0, 1.0, None)

        assert f(None, None, None) == 0 and f(p, p, None) == f(p, None, p) == f(None, p, None) == f(p + 4, None, None) == -4


def test_window_attention_refuses_a_scale_that_overflows():
    """in units of the kernels' powers of two the scale is 1.44 times larger: past 2.36e38 that is infinite, and every logit NaN"""
    with pytest.raises(RuntimeError, match="scale > 0"):
        ops.window_attention(X, X, X, 1, scale=2.5e38)
    buf = (ctypes.c_char * 512)()
    p = (ctypes.addressof(buf) + 63) // 64 * 64
    for suf in ("f32", "bf16"):
        f = getattr(hip.lib(), "indm_wattn_fwd_" + suf)
        strides = (ctypes.c_long * 9)(*[64] * 9)
        assert f(p, p, p, strides, p, None, None, None, 1, 4, 2, 1, 16, 1, 1, 0, 0, 2.5e38, None) == -4

"""Ways of calling the token operators that ask more of them than dense tensors do: lazily negated views, tensors of zeros without
memory, tensors that are not all on one device."""
import pytest
import torch
from torch.autograd import forward_ad

from indm_amd import hip, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SECTIONS = (8,)
NAMES = ["layer_norm", "dropout", "dropout res", "rotary", "rotary k", "q", "k", "v"]


def positions(T):
    return torch.arange(T, device=DEV)[:, None]


def operators(T=6, H=2, D=16):
    freqs, pos = ops.rotary_freqs(SECTIONS, device=DEV), positions(T)
    g = torch.Generator(device=DEV).manual_seed(1)
    other = torch.randn((2, T, H, D), generator=g, device=DEV)
    gamma = torch.randn((D,), generator=g, device=DEV)
    return {"layer_norm": lambda x: ops.layer_norm(x, gamma), "dropout": lambda x: ops.dropout(x, 0.4, 5), "dropout res": lambda x: ops.dropout(other, 0.4, 5, res=x),
            "rotary": lambda x: ops.rotary(x, None, pos, freqs, SECTIONS)[0], "rotary k": lambda x: ops.rotary(other, x, pos, freqs, SECTIONS)[1],
            "q": lambda x: ops.window_attention(x, other, other, 2), "k": lambda x: ops.window_attention(other, x, other, 2),
            "v": lambda x: ops.window_attention(other, other, x, 2)}


def negated(seed, shape=(2, 6, 2, 16)):
    """a view whose memory holds the negative of its values"""
    z = torch.randn(shape, dtype=torch.complex64, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).conj().imag
    assert z.is_neg()
    return z


@pytest.mark.parametrize("name", NAMES)
def test_negated_views_and_gradients(name):
    call, x, dy = operators()[name], negated(2), negated(3)
    plain = x.clone().requires_grad_()
    want = call(plain)
    (dwant,) = torch.autograd.grad(want, plain, dy.clone())
    with torch.no_grad():
        assert torch.equal(call(x), want)
    z = torch.complex(torch.zeros_like(plain), -plain.detach()).requires_grad_()
    view = z.conj().imag
    assert view.is_neg()
    got = call(view)
    (dz,) = torch.autograd.grad(got, z, dy)
    assert torch.equal(got, want) and torch.equal(dz.imag, -dwant)


@pytest.mark.parametrize("name", NAMES)
def test_zeros_without_memory(name):
    call = operators()[name]
    zero = torch._efficientzerotensor((2, 6, 2, 16), device=DEV)
    x = torch.zeros((2, 6, 2, 16), device=DEV)
    with torch.no_grad():
        assert torch.equal(call(zero), call(x))
    leaf = torch.randn((2, 6, 2, 16), device=DEV).requires_grad_()
    (g,) = torch.autograd.grad(call(leaf), leaf, zero)
    assert torch.equal(g, x)


def test_negated_parameters():
    x, p, n = negated(4).clone(), negated(5, (16,)), positions(6).to(torch.float32)
    neg_pos = torch.complex(torch.zeros_like(n), -n).conj().imag
    freqs = ops.rotary_freqs(SECTIONS, device=DEV)
    neg_freqs = torch.complex(torch.zeros_like(freqs), -freqs).conj().imag
    assert neg_pos.is_neg() and neg_freqs.is_neg()
    assert torch.equal(ops.layer_norm(x, p, p), ops.layer_norm(x, p.clone(), p.clone()))
    assert torch.equal(ops.rotary(x, None, neg_pos, neg_freqs, SECTIONS)[0], ops.rotary(x, None, n, freqs, SECTIONS)[0])


def test_tensors_left_on_the_host_are_refused():
    """a parameter, a residual, positions, lengths left on the host"""
    x, freqs, pos = torch.ones((2, 6, 2, 16), device=DEV), ops.rotary_freqs(SECTIONS, device=DEV), positions(6)
    for call in (lambda: ops.layer_norm(x, torch.ones(16)), lambda: ops.layer_norm(x, None, torch.ones(16)), lambda: ops.dropout(x, 0.5, 1, res=x.cpu()),
                 lambda: ops.rotary(x, x.cpu(), pos, freqs, SECTIONS), lambda: ops.rotary(x, None, pos.cpu(), freqs, SECTIONS),
                 lambda: ops.rotary(x, None, pos, freqs.cpu(), SECTIONS), lambda: ops.window_attention(x, x.cpu(), x, 2),
                 lambda: ops.window_attention(x, x, x, 2, lengths=torch.tensor([6, 6], dtype=torch.int32))):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


@pytest.mark.parametrize("C", [1, 3, 5, 64, 130, 300])
def test_layer_norm_of_large_constant_rows(C):
    """Rows of 2^119: -mean / sd overflows (2^119 / sqrt(1e-6) > 2^128) in the places behind a row that fill its last vector, and nothing of that
    may reach a gradient.  The sums are exact (up to 300 x 2^119 < 2^128); where C is a power of two the mean is, too: y = beta, dgamma = 0,
    dx = (h - mean h) / sqrt(eps).  Elsewhere the mean may be off by a step of 2^95, whose square overflows: sd is infinite, y = beta."""
    x = torch.full((4, C), 2.0 ** 119, device=DEV).requires_grad_()
    gamma, beta = torch.ones(C, device=DEV).requires_grad_(), torch.full((C,), 0.25, device=DEV).requires_grad_()
    dy = torch.randn((4, C), generator=torch.Generator(device=DEV).manual_seed(6), device=DEV)
    y = ops.layer_norm(x, gamma, beta)
    dx, dg, db = torch.autograd.grad(y, (x, gamma, beta), dy)
    assert (y == 0.25).all() and all(t.isfinite().all() for t in (dx, dg, db))
    if C & (C - 1) == 0:
        assert (dg == 0).all()
        want = (dy.double() - dy.double().mean(1, keepdim=True)) * 1e3
        # sums of at most 64 terms, half a step each; eps = 1e-6 in 32 bits, its root and its reciprocal
        assert ((dx.double() - want).abs() <= 80 * 2.0 ** -24 * 1e3 * dy.double().abs().sum(1, keepdim=True)).all()


def test_guard_bands_keep_their_own_size():
    """bands set anew, or switched off, between the call that made a tensor and the count: each tensor is counted by its own"""
    ext, x = hip.token_ops(), torch.ones(1000, device=DEV)
    try:
        for then in (1 << 16, 0):
            ext.guard(512)
            y = ops.dropout(x, 0.5, 1)
            ext.guard(then)
            assert ext.broken_guards() == 0
            ext.guard(512)
            y = ops.dropout(x, 0.5, 1)
            y.as_strided((1,), (1,), y.storage_offset() - 128).fill_(2.0)     # the first of the 128 floats in front of it
            ext.guard(then)
            assert ext.broken_guards() == 1 and ext.broken_guards() == 0
    finally:
        ext.broken_guards()
        ext.guard(0)


def test_guard_bands_while_other_threads_call():
    """calls on four threads, forward and backward, while the bands change: none is lost, none is counted by another's size"""
    import threading
    ext, bad = hip.token_ops(), []
    x = torch.randn((64, 96), device=DEV)
    want = ops.layer_norm(x)

    def work():
        try:
            for _ in range(50):
                leaf = x.clone().requires_grad_()
                y = ops.layer_norm(leaf)
                torch.autograd.grad(y, leaf, x)
                if not torch.equal(y, want):
                    bad.append("result")
        except Exception as e:   # noqa: BLE001
            bad.append(e)

    threads = [threading.Thread(target=work) for _ in range(4)]
    try:
        for t in threads:
            t.start()
        for i in range(200):
            ext.guard((0, 256, 1 << 14)[i % 3])
        for t in threads:
            t.join()
        assert not bad and ext.broken_guards() == 0
    finally:
        ext.broken_guards()
        ext.guard(0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,T,H,Hk", [(1, 90, 2, 1), (1, 500, 8, 2), (5, 600, 8, 2), (40, 300, 4, 4)])     # (each layout of the key kernels)
def test_window_attention_wanted_gradients_only(dtype, B, T, H, Hk):
    """some of q, k, v frozen: the others' gradients are the same numbers"""
    g = torch.Generator(device=DEV).manual_seed(7)
    xs = [torch.randn((B, T, h, 32), generator=g, device=DEV).to(dtype) for h in (H, Hk, Hk)]
    do = torch.randn((B, T, H, 32), generator=g, device=DEV).to(dtype)
    lengths = torch.tensor([T - b % 3 * 17 for b in range(B)], dtype=torch.int32, device=DEV)

    def grads(keep):
        leaves = [x.clone().requires_grad_(i in keep) for i, x in enumerate(xs)]
        o = ops.window_attention(*leaves, 200, sinks=3, lengths=lengths)
        return torch.autograd.grad(o, [leaves[i] for i in keep], do)

    want = grads((0, 1, 2))
    for keep in ((0,), (1,), (2,), (0, 1), (1, 2), (0, 2)):
        assert all(torch.equal(a, want[i]) for a, i in zip(grads(keep), keep)), keep


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R,C", [(50, 96), (9000, 256), (300, 1153), (40, 9000)])
def test_layer_norm_parameters_alone(dtype, R, C):
    """x frozen: no gradient of it is made, and the parameters' are the same numbers"""
    g = torch.Generator(device=DEV).manual_seed(8)
    x, dy = (torch.randn((R, C), generator=g, device=DEV).to(dtype) for _ in range(2))
    gamma, beta = (torch.randn((C,), generator=g, device=DEV).requires_grad_() for _ in range(2))
    leaf = x.clone().requires_grad_()
    want = torch.autograd.grad(ops.layer_norm(leaf, gamma, beta), (gamma, beta), dy)
    y = ops.layer_norm(x, gamma, beta)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    got = torch.autograd.grad(y, (gamma, beta), dy)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    if R * C > 1 << 21:     # (its partial sums take 16 bytes a column of up to 1024 workgroups' rows)
        assert torch.cuda.max_memory_allocated() - before < x.numel() * x.element_size() + 8 * C * min(R, 1024)


@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_through_a_backward_pass_is_refused(name):
    """a gradient with a tangent: that of the result would be lost without a word"""
    call, leaf, dy = operators()[name], torch.randn((2, 6, 2, 16), device=DEV).requires_grad_(), torch.randn((2, 6, 2, 16), device=DEV)
    y = call(leaf)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(dy, dy)
        if name == "dropout res":      # (its gradient is the one that came in, with its tangent)
            (g,) = torch.autograd.grad(y, leaf, dual, retain_graph=True)
            assert torch.equal(forward_ad.unpack_dual(g).tangent, dy)
        else:
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(y, leaf, dual, retain_graph=True)
    (g,) = torch.autograd.grad(y, leaf, dy)
    assert g.isfinite().all()

"""Window attention with sinks (csrc/window_attn.hip) against its definition in 64 bits, forward and gradients, with guard bands
around every allocation of the package.

Tolerances count roundings, u = 2^-24, h = half a step of the tensors' type (bf16 2^-8, fp32 2^-24).
  logits   z = scale q.k: D products and sums in fp32: (D + 4) u scale |q|.|k|; the exponent adds 2 u |z| + 2 u |lse|, exp2 and the row's
           sum of N terms 8 u + N u.  P is off by that relative error E (its own and, through the sum, its row's largest: 2 max E).
  o        sum P v: each P rounded to an operand (h), N fp32 sums, one rounding of the result
  dS       P (dP - delta): dP is D products, delta = <do, o> takes o as it was stored
  dq, dk   sums of dS k, dS q with dS rounded to an operand;  dv  sum P do"""
import math

import pytest
import torch

from indm_amd import hip, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
DTYPES = [torch.float32, torch.bfloat16]


@pytest.fixture
def guards():
    """guard bands of 64 KB around every tensor that the kernels write"""
    ext = hip.token_ops()
    ext.guard(1 << 16)
    try:
        yield ext
    finally:
        ext.broken_guards()
        ext.guard(0)


def randn(shape, seed, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV) * scale).to(dtype)


def visible(T, left, right, sinks, causal, n):
    i = torch.arange(T, device=DEV)[:, None]
    j = torch.arange(T, device=DEV)[None, :]
    m = ((j >= i - left) & (j <= i + right)) | (j < sinks)
    if causal:
        m = m & (j <= i)
    return m & (i < n) & (j < n)


def reference(q, k, v, do, left, right, sinks, causal, lengths, scale):
    """-> (o, dq, dk, dv) and a bound for each, in 64 bits"""
    B, T, H, D = q.shape
    Hk = k.shape[2]
    h = HALF[q.dtype]
    q64, k64, v64, do64 = (x.double() for x in (q, k, v, do))
    out = [torch.zeros_like(x) for x in (q64, q64, k64, v64)]
    tol = [torch.zeros_like(x) for x in (q64, q64, k64, v64)]
    for b in range(B):
        n = T if lengths is None else max(0, min(T, int(lengths[b])))
        if n == 0:
            continue
        see = visible(T, left, right, sinks, causal, n)[:n, :n]
        N = int(see.sum(1).max())
        Nk = int(see.sum(0).max()) * (H // Hk)
        for hh in range(H):
            g = hh // (H // Hk)
            Q, K, V, dO = q64[b, :n, hh], k64[b, :n, g], v64[b, :n, g], do64[b, :n, hh]
            mm = lambda a, c: a @ c.contiguous()  # noqa: E731
            z = mm(Q, K.t()) * scale
            zm = z.masked_fill(~see, -math.inf)
            lse = zm.logsumexp(1, keepdim=True)
            P = torch.exp(zm - lse)
            O = mm(P, V)
            E = U * ((D + 4) * scale * mm(Q.abs(), K.abs().t()) + 2 * z.abs() + 2 * lse.abs() + 8 + N)
            E = 2 * E.masked_fill(~see, 0.0).amax(1, keepdim=True)
            eo = mm(P, V.abs()) * (h + E + (N + 4) * U) + h * O.abs()
            out[0][b, :n, hh], tol[0][b, :n, hh] = O, eo
            dP = mm(dO, V.t())
            delta = (dO * O).sum(1, keepdim=True)
            dS = P * (dP - delta)
            edP = (D + 4) * U * mm(dO.abs(), V.abs().t())
            edelta = (dO.abs() * eo).sum(1, keepdim=True) + (D + 4) * U * (dO * O).abs().sum(1, keepdim=True)
            eS = dS.abs() * (h + E + 4 * U) + P * (edP + edelta)
            dq = scale * mm(dS, K)
            out[1][b, :n, hh] = dq
            tol[1][b, :n, hh] = scale * (mm(eS, K.abs()) + (N + 8) * U * mm(dS.abs(), K.abs())) + (h + 2 * U) * dq.abs()
            out[2][b, :n, g] += scale * mm(dS.t().contiguous(), Q)
            tol[2][b, :n, g] += scale * (mm(eS.t().contiguous(), Q.abs()) + (Nk + 8) * U * mm(dS.abs().t().contiguous(), Q.abs()))
            out[3][b, :n, g] += mm(P.t().contiguous(), dO)
            tol[3][b, :n, g] += mm((P * (h + E + (Nk + 8) * U)).t().contiguous(), dO.abs())
    for i in (2, 3):
        tol[i] += (h + 2 * U) * out[i].abs()
    return out, tol


def close(got, want, tol, what):
    d = (got.double() - want).abs()
    bad = ~(d <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}, worst {float((d - tol)[bad].max())} over"


def check(q, k, v, do, left, right, sinks=0, causal=False, lengths=None, scale=None, window="pair"):
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    o = ops.window_attention(*leaves, (left, right), sinks=sinks, causal=causal, lengths=lengths, scale=scale)
    grads = torch.autograd.grad(o, leaves, do)
    assert o.dtype == q.dtype and o.shape == q.shape and all(g.shape == x.shape and g.dtype == x.dtype for g, x in zip(grads, leaves))
    with torch.no_grad():
        assert torch.equal(ops.window_attention(*leaves, (left, right), sinks=sinks, causal=causal, lengths=lengths, scale=scale), o)
    T, far = q.shape[1], q.shape[1]
    clean = [x.detach() for x in (q, k, v, do)]
    if lengths is not None:     # what lies behind a sequence is nobody's: the reference does not look at it
        dead = torch.arange(T, device=DEV)[None, :] >= lengths.clamp(0, T)[:, None]
        clean = [x.masked_fill(dead[:, :, None, None], 0.0) for x in clean]
    want, tol = reference(*clean, far if left is None else left, far if right is None else right, sinks, causal, lengths,
                          q.shape[-1] ** -0.5 if scale is None else scale)
    for name, got, w, e in zip(("o", "dq", "dk", "dv"), (o.detach(), *grads), want, tol):
        close(got, w, e, name)
        if lengths is not None:
            assert (got[dead] == 0).all(), name


CASES = [  # B, T, H, Hk, D, left, right, sinks, causal
    (1, 1, 1, 1, 8, 0, 0, 0, False), (2, 2, 2, 1, 16, 1, 0, 0, True), (1, 3, 1, 1, 32, 0, 0, 1, False), (1, 31, 2, 2, 64, 4, 7, 2, False),
    (2, 32, 1, 1, 32, 32, 32, 0, False), (1, 33, 3, 1, 24, 5, 5, 0, False), (1, 63, 2, 1, 40, 9, 0, 3, True), (1, 64, 2, 2, 128, 64, 64, 0, False),
    (1, 65, 4, 2, 64, 16, 16, 1, False), (2, 127, 2, 1, 72, 20, 3, 5, False), (1, 128, 2, 2, 96, 31, 0, 4, True), (1, 129, 2, 1, 104, 3, 64, 33, False),
    (1, 300, 6, 2, 64, 40, 40, 4, False), (1, 300, 2, 2, 64, 40, 0, 4, True), (2, 257, 4, 1, 128, 100, 1, 70, False), (1, 1000, 2, 1, 64, 64, 64, 1, False),
    (1, 1000, 3, 3, 32, 7, 250, 16, False), (1, 777, 2, 1, 64, None, None, 0, False), (1, 777, 2, 1, 64, None, None, 0, True),
    (1, 500, 1, 1, 64, None, 5, 9, False), (1, 500, 1, 1, 64, 5, None, 9, False), (1, 400, 2, 1, 64, 0, 0, 0, False), (1, 400, 2, 1, 64, 0, 0, 2, True),
    (1, 200, 2, 1, 64, 3, 3, 500, False), (1, 200, 2, 1, 64, 3, 3, 150, True), (3, 1100, 8, 2, 16, 70, 30, 2, False), (1, 2500, 1, 1, 128, 128, 0, 40, True)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", CASES)
def test_sizes_and_windows(guards, dtype, case):
    B, T, H, Hk, D, left, right, sinks, causal = case
    q, k, v, do = (randn((B, T, h, D), 1 + i, dtype, 1.3 if i < 2 else 1.0) for i, h in enumerate((H, Hk, Hk, H)))
    check(q, k, v, do, left, right, sinks, causal)
    assert guards.broken_guards() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("B,T,H,Hk,D,left,right,sinks", [
    (40, 300, 4, 4, 32, 30, 20, 5),       # key blocks that fill the chip: the sinks' queries in a launch of their own
    (40, 300, 4, 4, 32, 3, 2, 200),       # the same with several blocks of sinks
    (5, 600, 8, 2, 64, 300, 100, 16),     # key blocks whose queries are split, the sinks' workgroups behind them
    (5, 600, 8, 2, 64, 300, 100, 290)])
def test_workgroup_layouts(guards, dtype, causal, B, T, H, Hk, D, left, right, sinks):
    """the backward pass' layouts that small cases do not reach, with sequences that end among the sinks and an empty one"""
    q, k, v, do = (randn((B, T, h, D), 130 + i, dtype) for i, h in enumerate((H, Hk, Hk, H)))
    lengths = torch.tensor([T, 0, sinks // 2, T - 1, 129] * (B // 5), dtype=torch.int32, device=DEV)
    check(q, k, v, do, left, right, sinks, causal, lengths)
    assert guards.broken_guards() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [8, 16, 32, 48, 64, 80, 96, 112, 120, 128])
def test_head_widths(guards, dtype, D):
    q, k, v, do = (randn((1, 150, h, D), 10 + i, dtype) for i, h in enumerate((2, 1, 1, 2)))
    check(q, k, v, do, 30, 30, 2, scale=0.3)
    assert guards.broken_guards() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("T,ns", [(70, [70, 0, 1, 33, 64, 65, 200, -3]), (300, [300, 129, 128, 127, 2]), (5, [0, 0]), (130, [0, 130])])
def test_lengths(guards, dtype, causal, T, ns):
    """sequences of every length, none and all; what lies behind them is NaN or infinite and must not show anywhere"""
    B = len(ns)
    lengths = torch.tensor(ns, dtype=torch.int32, device=DEV)
    xs = [randn((B, T, h, 64), 20 + i, dtype) for i, h in enumerate((2, 1, 1, 2))]
    dead = torch.arange(T, device=DEV)[None, :] >= lengths[:, None]
    for x, bad in zip(xs, (math.nan, math.inf, -math.inf, math.nan)):
        x[dead] = bad
    check(*xs, 20, 10, 3, causal, lengths)
    assert guards.broken_guards() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("how", ["fused product", "odd offset", "heads first", "columns not contiguous", "shared by the batch"])
def test_strides(guards, dtype, how):
    B, T, H, Hk, D = 2, 90, 4, 2, 40
    if how in ("fused product", "odd offset"):
        o = 0 if how == "fused product" else 3
        qkv = randn((B, T, (H + 2 * Hk) * D + 8), 30, dtype)
        q, k, v = (qkv[..., o + a * D:o + b * D].unflatten(-1, (b - a, D)) for a, b in ((0, H), (H, H + Hk), (H + Hk, H + 2 * Hk)))
    elif how == "heads first":
        q, k, v = (randn((B, h, T, D), 31 + i, dtype).transpose(1, 2) for i, h in enumerate((H, Hk, Hk)))
    elif how == "columns not contiguous":
        q, k, v = (randn((B, T, D, h), 34 + i, dtype).transpose(2, 3) for i, h in enumerate((H, Hk, Hk)))
    else:
        q, k, v = randn((B, T, H, D), 37, dtype), randn((1, T, Hk, D), 38, dtype).expand(B, -1, -1, -1), randn((B, T, 1, D), 39, dtype).expand(-1, -1, Hk, -1)
    do = randn((B, T, 1, D), 40, dtype).expand(-1, -1, H, -1)     # a broadcast gradient
    check(q, k, v, do, 25, 12, 2)
    assert guards.broken_guards() == 0


def test_offsets_past_32_bits():
    """more than 2^31 elements in every tensor: the last tokens against the definition on the tokens that they reach"""
    T, H, D, n = 140_000, 124, 128, 40
    xs = [torch.zeros((1, T, H, D), dtype=torch.bfloat16, device=DEV) for _ in range(4)]
    for i, x in enumerate(xs):
        x[:, -n:] = randn((1, n, H, D), 110 + i, torch.bfloat16)
    leaves = [x.requires_grad_() for x in xs[:3]]
    o = ops.window_attention(*leaves, (n, 0))
    grads = torch.autograd.grad(o, leaves, xs[3])
    want, tol = reference(*(x.detach()[:, -2 * n:] for x in xs), n, 0, 0, False, None, D ** -0.5)
    for name, got, w, e in zip(("o", "dq", "dk", "dv"), (o.detach(), *grads), want, tol):
        close(got[:, -n:], w[:, -n:], e[:, -n:], name)
    assert (o.detach()[:, :-2 * n:997] == 0).all() and (grads[2][:, :-2 * n:997] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_what_is_not_finite_stays_near(dtype):
    """a token of NaN leaves the rows beyond its window and 64 more as they are, bit for bit"""
    T, w, at = 600, 20, 333
    xs = [randn((1, T, h, 64), 120 + i, dtype) for i, h in enumerate((4, 2, 2, 4))]
    runs = []
    for bad in (False, True):
        leaves = [x.clone() for x in xs]
        if bad:
            for x in leaves:
                x[:, at] = math.nan
        *qkv, do = leaves
        qkv = [x.requires_grad_() for x in qkv]
        o = ops.window_attention(*qkv, w, sinks=3)
        runs.append((o.detach(), *torch.autograd.grad(o, qkv, do)))
    far = (torch.arange(T, device=DEV) - at).abs() > w + 64
    sinks = torch.arange(T, device=DEV) < 3      # (they gather from every query: their dk and dv)
    for clean, got in zip(*runs):
        assert torch.equal(clean[:, far & ~sinks], got[:, far & ~sinks])


def test_large_logits_keep_the_row_maximum():
    """logits of several hundred, growing along the keys, so that the running maximum has to be raised again and again"""
    T = 500
    q, v, do = (randn((1, T, 1, 64), 41 + i) for i in range(3))
    k = q.mean(1, keepdim=True) + randn((1, T, 1, 64), 44) * torch.linspace(0.1, 12.0, T, device=DEV)[None, :, None, None]
    check(q * 4, k, v, do, None, None)
    check((q * 4).bfloat16(), k.bfloat16(), v.bfloat16(), do.bfloat16(), None, None)


def test_one_visible_key_is_copied():
    """a window of nothing but the token itself: o = v, dv = do, and the softmax has no slope"""
    q, k, v, do = (randn((2, 77, 2, 32), 45 + i) for i in range(4))
    leaves = [x.requires_grad_() for x in (q, k, v)]
    o = ops.window_attention(*leaves, 0)
    dq, dk, dv = torch.autograd.grad(o, leaves, do)
    # the one logit and its maximum are below 8: their exponent is 0 but for u 8 on each side of the difference, P / P is 1
    assert ((o - v).abs() <= 16 * U * v.abs()).all() and ((dv - do).abs() <= 32 * U * do.abs()).all()
    # dS = dP - delta of two sums of the same 32 products: 36 u of them each, and 48 u for o's own error
    slack = 120 * U * (do.abs() * v.abs()).sum(-1, keepdim=True) * 32 ** -0.5
    assert (dq.abs() <= slack * k.abs() * 1.01).all() and (dk.abs() <= slack * q.abs() * 1.01).all()


def test_window_forms():
    q, k, v = (randn((1, 60, 2, 32), 50 + i) for i in range(3))
    f = lambda *a, **kw: ops.window_attention(q, k, v, *a, **kw)  # noqa: E731
    assert torch.equal(f(7), f((7, 7))) and torch.equal(f(), f((60, 60))) and torch.equal(f((None, 0)), f(causal=True))
    assert torch.equal(f((10 ** 12, 3)), f((None, 3))) and torch.equal(f(5, causal=True), f((5, 0)))
    assert torch.equal(f(3, sinks=10 ** 9), f())


@pytest.mark.parametrize("B,T,H", [(0, 5, 2), (2, 0, 2)])
def test_empty(B, T, H):
    q, k, v = (torch.zeros((B, T, H, 16), device=DEV, requires_grad=True) for _ in range(3))
    o = ops.window_attention(q, k, v, 3, sinks=1)
    g = torch.autograd.grad(o, (q, k, v), torch.zeros_like(o))
    assert o.shape == g[0].shape == g[2].shape == (B, T, H, 16)


@pytest.mark.parametrize("dtype", DTYPES)
def test_same_bits(dtype):
    xs = [randn((2, 700, h, 64), 60 + i, dtype) for i, h in enumerate((4, 2, 2, 4))]
    ref = None
    for _ in range(3):
        leaves = [x.clone().requires_grad_() for x in xs[:3]]
        o = ops.window_attention(*leaves, (90, 60), sinks=40)
        got = (o.detach(), *torch.autograd.grad(o, leaves, xs[3]))
        assert ref is None or all(torch.equal(a, b) for a, b in zip(ref, got))
        ref = got


def test_gradient_against_differences():
    """central differences of the kernel's own forward pass: step 2^-6, truncation s^2/6 of a third derivative of some tens (a few
    1e-3), rounding 2 u |f| / s with |f| < 300 (2e-3)"""
    xs = [randn((1, 40, h, 16), 70 + i) for i, h in enumerate((2, 1, 1))]
    w = randn((1, 40, 2, 16), 73)
    kw = dict(window=(9, 5), sinks=2)
    leaves = [x.clone().requires_grad_() for x in xs]
    grads = torch.autograd.grad(ops.window_attention(*leaves, **kw), leaves, w)
    f = lambda *v: float((ops.window_attention(*v, **kw).double() * w.double()).sum())  # noqa: E731
    s = 2.0 ** -6
    for i in range(3):
        d = randn(xs[i].shape, 74 + i, scale=0.5)
        up, down = list(xs), list(xs)
        up[i], down[i] = up[i] + s * d, down[i] - s * d
        assert abs((f(*up) - f(*down)) / (2 * s) - float((grads[i].double() * d.double()).sum())) < 0.02, i


def test_second_derivatives_are_refused():
    q, k, v = (randn((1, 8, 1, 16), 80 + i).requires_grad_() for i in range(3))
    (g,) = torch.autograd.grad(ops.window_attention(q, k, v, 2).square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_streams_and_captured_graphs():
    """two streams at once, and two captured graphs that replay in turn with eager work between: always the eager bits"""
    xs = [randn((2, 333, h, 64), 90 + i, torch.bfloat16) for i, h in enumerate((4, 2, 2, 4))]
    lengths = torch.tensor([333, 200], dtype=torch.int32, device=DEV)

    def step(window):
        leaves = [x.detach().requires_grad_() for x in xs[:3]]
        o = ops.window_attention(*leaves, window, sinks=3, lengths=lengths)
        return [o.detach(), *torch.autograd.grad(o, leaves, xs[3])]

    want = step(50)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [None, None]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = step(50)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))
    graphs = []
    for window in (50, 17):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(window)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(window)
        graphs.append((window, g, out))
    for rep in range(3):
        for i, x in enumerate(xs):
            x.copy_(randn(x.shape, 100 + 10 * rep + i, torch.bfloat16))
        lengths.copy_(torch.tensor([100 + rep, 333 - rep], dtype=torch.int32))
        for window, g, out in graphs:
            want = step(window)
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want)), (rep, window)

"""Layer norm, dropout and rotary positions (csrc/token_ops.hip) against their definitions in 64 bits, at the sizes, strides and
values where they can go wrong, with guard bands around every allocation of the package.

Tolerances count roundings.  u = 2^-24 is half a step of fp32, h = half a step of the result's type (bf16 2^-8, fp32 2^-24).
A value v that is computed in fp32 and rounded once is off by at most h |v| plus what its fp32 terms have gathered; each bound
below names those terms."""
import math

import numpy as np
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


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(shape, seed, dtype=torch.float32, scale=1.0, mean=0.0):
    return (torch.randn(shape, generator=gen(seed), device=DEV) * scale + mean).to(dtype)


def close(got, want, tol, what=""):
    """|got - want| <= tol everywhere (tol: a tensor or a number)"""
    d = (got.double() - want).abs()
    bad = ~(d <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((d - tol)[bad].max())} over its bound"


def test_guard_bands_catch_an_overrun(guards):
    y = ops.dropout(torch.ones(1000, device=DEV), 0.5, 1)
    assert guards.broken_guards() == 0
    y = ops.dropout(torch.ones(1000, device=DEV), 0.5, 1)
    y.as_strided((1,), (1,), 1000 + y.storage_offset()).fill_(2.0)     # one element past the end
    assert guards.broken_guards() == 1


# ---------------------------------------------------------------------------------------------- layer norm
# every team of the kernels (16 ... 1024 lanes) at and around its last width, one row to many, odd widths and row counts
LN_SHAPES = [(1, 1), (3, 1), (1, 2), (7, 5), (5, 64), (300, 65), (17, 128), (9, 129), (257, 256), (33, 257), (64, 512), (31, 513), (5, 1024),
             (6, 1025), (12, 1153), (3, 2048), (4, 2049), (3, 4096), (2, 4099), (2, 8192), (1, 16384), (2, 16383), (4200, 48), (2065, 256)]


def ln_reference(x, gamma, beta, eps, dy):
    x, dy = x.double(), dy.double()
    C = x.shape[-1]
    g = torch.ones(C, dtype=torch.float64, device=x.device) if gamma is None else gamma.double()
    b = 0.0 if beta is None else beta.double()
    m = x.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt(((x - m) ** 2).mean(-1, keepdim=True) + eps)
    xh = (x - m) * rstd
    h = dy * g
    dx = rstd * (h - h.mean(-1, keepdim=True) - xh * (h * xh).mean(-1, keepdim=True))
    return xh * g + b, dx, (dy * xh), dy, xh, rstd, g


def ln_check(x, gamma, beta, eps, dy, y, dx, dg, db):
    want_y, want_dx, tg, tb, xh, rstd, g = ln_reference(x, gamma, beta, eps, dy)
    h = HALF[x.dtype]
    C, R = x.shape[-1], x.numel() // x.shape[-1]
    # the longest chain of additions of a row's sums: at most 32 elements a lane, 6 shuffles, then the wavefronts (4) -- 48 with
    # the products; the row's mean carries that error times mean |x|, the variance's relative error is as much, halved by the root
    n = 48
    amax = x.double().abs().amax(-1, keepdim=True)
    err_xh = U * ((n + 2) * amax * rstd + (n + 4) * xh.abs())
    close(y, want_y, h * want_y.abs() + (err_xh + 2 * U * xh.abs()) * g.abs() + 2 * U * want_y.abs(), "y")
    if dx is not None:
        hv = (dy.double() * g).abs()
        # dx's three terms: each mean carries n roundings of its summands, and the error of xh where it enters
        mean_h, mean_hx = hv.mean(-1, keepdim=True), (hv * xh.abs()).mean(-1, keepdim=True)
        e = U * (4 * hv + (n + 4) * mean_h + (n + 6) * xh.abs() * mean_hx) + err_xh * mean_hx + xh.abs() * (hv * err_xh).mean(-1, keepdim=True)
        rel_rstd = U * (n + 4 + (n + 2) * amax * rstd)
        close(dx, want_dx, h * want_dx.abs() + rstd * e + rel_rstd * want_dx.abs() + 2 * U * want_dx.abs(), "dx")
    # columns: a team adds its rows one after another (at most R of them here), then teams, workgroups and runs are joined
    chain = min(R, 4096) + 64
    if dg is not None:
        close(dg, tg.reshape(-1, C).sum(0), (U * chain * tg.abs() + err_xh * dy.double().abs()).reshape(-1, C).sum(0), "dgamma")
    if db is not None:
        close(db, tb.reshape(-1, C).sum(0), (U * chain * tb.abs()).reshape(-1, C).sum(0), "dbeta")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,C", LN_SHAPES)
def test_layer_norm_sizes(guards, dtype, R, C):
    x = randn((R, C), 1, dtype, 2.0, 0.4).requires_grad_()
    gamma, beta = randn((C,), 2, scale=0.3, mean=1.0).requires_grad_(), randn((C,), 3).requires_grad_()
    dy = randn((R, C), 4, dtype)
    y = ops.layer_norm(x, gamma, beta)
    dx, dg, db = torch.autograd.grad(y, (x, gamma, beta), dy)
    assert y.dtype == dx.dtype == dtype and dg.dtype == db.dtype == torch.float32
    ln_check(x.detach(), gamma.detach(), beta.detach(), 1e-6, dy, y.detach(), dx, dg, db)
    with torch.no_grad():
        assert torch.equal(ops.layer_norm(x, gamma, beta), y)
    assert guards.broken_guards() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("affine", ["none", "gamma", "beta"])
def test_layer_norm_without_parameters(guards, dtype, affine):
    x = randn((37, 200), 5, dtype).requires_grad_()
    gamma = randn((200,), 6, mean=1.0).requires_grad_() if affine == "gamma" else None
    beta = randn((200,), 7).requires_grad_() if affine == "beta" else None
    dy = randn((37, 200), 8, dtype)
    y = ops.layer_norm(x, gamma, beta, eps=1e-3)
    leaves = [v for v in (x, gamma, beta) if v is not None]
    g = torch.autograd.grad(y, leaves, dy)
    ln_check(x.detach(), None if gamma is None else gamma.detach(), None if beta is None else beta.detach(), 1e-3, dy, y.detach(), g[0],
             g[1] if affine == "gamma" else None, g[1] if affine == "beta" else None)
    assert guards.broken_guards() == 0


def test_layer_norm_wanted_gradients_only(guards):
    """frozen input or parameters: the other gradients are the same numbers"""
    x, gamma, beta, dy = randn((50, 96), 9), randn((96,), 10), randn((96,), 11), randn((50, 96), 12)
    full = [v.clone().requires_grad_() for v in (x, gamma, beta)]
    want = torch.autograd.grad(ops.layer_norm(*full), full, dy)
    for keep in range(3):
        some = [v.clone().requires_grad_(i == keep) for i, v in enumerate((x, gamma, beta))]
        (got,) = torch.autograd.grad(ops.layer_norm(*some), [some[keep]], dy)
        assert torch.equal(got, want[keep])
    assert guards.broken_guards() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("how", ["slice", "odd slice", "3-d slice", "transposed", "every second", "expanded rows", "one column"])
def test_layer_norm_strides(guards, dtype, how):
    base = randn((24, 40, 130), 13, dtype)
    x = {"slice": base[0, :, 8:120], "odd slice": base[0, :, 3:116], "3-d slice": base[..., 1:98], "transposed": base.transpose(1, 2),
         "every second": base[..., ::2], "expanded rows": base[0, :1, :].expand(40, 130), "one column": base[0, :, 5:6]}[how].requires_grad_()
    C = x.shape[-1]
    gamma, beta = randn((2 * C,), 14)[::2].requires_grad_(), randn((C,), 15).requires_grad_()
    dy = randn((C,), 16, dtype).expand(x.shape)      # a broadcast gradient
    y = ops.layer_norm(x, gamma, beta)
    dx, dg, db = torch.autograd.grad(y, (x, gamma, beta), dy)
    ln_check(x.detach(), gamma.detach(), beta.detach(), 1e-6, dy, y.detach(), dx, dg, db)
    assert guards.broken_guards() == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_norm_empty_rows(dtype):
    x = torch.zeros((0, 64), dtype=dtype, device=DEV, requires_grad=True)
    gamma = torch.ones(64, device=DEV, requires_grad=True)
    y = ops.layer_norm(x, gamma)
    dx, dg = torch.autograd.grad(y, (x, gamma), torch.zeros_like(y))
    assert y.shape == dx.shape == (0, 64) and torch.equal(dg, torch.zeros_like(dg))


def test_layer_norm_offset_rows_keep_their_variance():
    """a mean 4096 times the spread: the squared differences are taken from the mean, not as a difference of large sums"""
    x = (randn((64, 320), 17).double() + 4096.0).float()
    y = ops.layer_norm(x)
    want = ln_reference(x, None, None, 1e-6, torch.zeros_like(x))[0]
    # the mean is within 48 u 4096 < 0.012 ... of which every difference carries the same part: that, against a spread of one
    close(y, want, 48 * U * 4100 + 60 * U * 5, "y")


def test_layer_norm_offsets_past_32_bits():
    """2^31 and more elements: the last rows come out as those rows alone do, and their gradients"""
    R, C = (1 << 22) + 5, 520
    x = torch.zeros((R, C), dtype=torch.bfloat16, device=DEV)
    x[-9:] = randn((9, C), 90, torch.bfloat16, 2.0, 1.0)
    x.requires_grad_()
    dy = torch.zeros((R, C), dtype=torch.bfloat16, device=DEV)
    dy[-9:] = randn((9, C), 91, torch.bfloat16)
    tail, dtail = x.detach()[-9:].clone().requires_grad_(), dy[-9:].clone()
    y, yt = ops.layer_norm(x), ops.layer_norm(tail)
    assert torch.equal(y[-9:], yt) and (y[:-9:100_003] == 0).all()
    (g,), (gt,) = torch.autograd.grad(y, x, dy), torch.autograd.grad(yt, tail, dtail)
    assert torch.equal(g[-9:], gt) and (g[:-9:100_003] == 0).all()


def test_layer_norm_infinities_stay_in_their_rows():
    x = randn((6, 96), 18)
    clean = ops.layer_norm(x)
    x[1, 3], x[4, 95] = math.inf, math.nan
    y = ops.layer_norm(x)
    for r in range(6):
        assert (y[r].isnan().all() if r in (1, 4) else torch.equal(y[r], clean[r]))


@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_norm_same_bits(dtype):
    x, dy = randn((5000, 320), 19, dtype).requires_grad_(), randn((5000, 320), 20, dtype)
    gamma = randn((320,), 21).requires_grad_()
    ref = None
    for _ in range(3):
        y = ops.layer_norm(x, gamma)
        got = (y, *torch.autograd.grad(y, (x, gamma), dy))
        assert ref is None or all(torch.equal(a, b) for a, b in zip(ref, got))
        ref = got


def test_layer_norm_gradient_against_differences():
    """directional central differences of the kernel's own forward pass, step s = 2^-6: the truncation is s^2 / 6 times the third
    derivative along a unit-size direction (a few tens here), the rounding 2 u |f| / s with |f| < 300: 0.02 together, of about 10"""
    x, gamma, beta = randn((12, 40), 22), randn((40,), 23, mean=1.0), randn((40,), 24)
    w = randn((12, 40), 25)
    leaves = [v.clone().requires_grad_() for v in (x, gamma, beta)]
    grads = torch.autograd.grad(ops.layer_norm(*leaves), leaves, w)
    f = lambda *v: float((ops.layer_norm(*v).double() * w.double()).sum())  # noqa: E731
    s = 2.0 ** -6
    for i in range(3):
        d = randn(leaves[i].shape, 26 + i, scale=0.5)
        up, down = [x, gamma, beta], [x, gamma, beta]
        up[i], down[i] = up[i] + s * d, down[i] - s * d
        assert abs((f(*up) - f(*down)) / (2 * s) - float((grads[i].double() * d.double()).sum())) < 0.02


# ---------------------------------------------------------------------------------------------- dropout
def philox_keep(seed, n, p):
    """the mask's definition, on the host in unsigned 64-bit words"""
    m = np.uint64(0xFFFFFFFF)
    c = [np.arange((n + 3) // 4, dtype=np.uint64)]
    c = [c[0] & m, c[0] >> np.uint64(32)] + [np.zeros_like(c[0]) for _ in range(2)]
    k = [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & m, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & m]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    w = np.stack(c, -1).reshape(-1)[:n]
    return torch.from_numpy(((w >> np.uint64(8)).astype(np.float64) + 1.0) * 2.0 ** -24 > float(np.float32(p))).to(DEV)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 7, 8, 9, 255, 1000, 4099, 300_001])
@pytest.mark.parametrize("residual", [False, True])
def test_dropout_sizes(guards, dtype, n, residual):
    p, seed = 0.3, 0x1234_5678_9ABC_DEF0 + n
    x = randn((n,), 30, dtype).requires_grad_()
    res = randn((n,), 31, dtype).requires_grad_() if residual else None
    dy = randn((n,), 32, dtype)
    y = ops.dropout(x, p, seed, res)
    g = torch.autograd.grad(y, [x] + ([res] if residual else []), dy)
    keep = philox_keep(seed, n, p)
    h = HALF[dtype]
    scaled = keep * x.detach().double() / (1 - float(np.float32(p)))
    want = scaled + (res.detach().double() if residual else 0.0)
    # the factor is off by two half steps, its product by one, the sum by one more
    close(y.detach(), want, h * want.abs() + U * (3 * scaled.abs() + want.abs()), "y")
    dwant = keep * dy.double() / (1 - float(np.float32(p)))
    close(g[0], dwant, h * dwant.abs() + 3 * U * dwant.abs(), "dx")
    assert (y.detach()[~keep] == (res.detach()[~keep] if residual else 0.0)).all() and (g[0][~keep] == 0).all()
    if residual:
        assert torch.equal(g[1], dy)
    assert guards.broken_guards() == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_dropout_mask_is_group_norms(dtype):
    """the same seed drops the same elements as the fused GroupNorm + dropout"""
    x = randn((2, 8, 8, 64), 33, dtype, mean=5.0)
    gamma, beta = torch.ones(64, device=DEV), torch.full((64,), 50.0, device=DEV)   # (no normalised value is zero)
    a = ops.group_norm(x, gamma, beta, drop_p=0.25, seed=77)
    b = ops.dropout(x, 0.25, 77)
    assert torch.equal(a == 0, b == 0) and 0.2 < float((b == 0).float().mean()) < 0.3


@pytest.mark.parametrize("dtype", DTYPES)
def test_dropout_edges(dtype):
    x = randn((1000,), 34, dtype)
    assert torch.equal(ops.dropout(x, 0.0, 5), x)
    assert (ops.dropout(x, 1.0, 5) == 0).all()
    assert torch.equal(ops.dropout(x, 1.0, 5, res=x), x)
    assert ops.dropout(x[:0], 0.5, 5).shape == (0,)
    bad = torch.full((1000,), math.nan, dtype=dtype, device=DEV)
    bad[::2] = -math.inf
    y = ops.dropout(bad, 0.5, 6)
    keep = philox_keep(6, 1000, 0.5)
    assert (y[~keep] == 0).all() and torch.equal(y[keep].isnan(), bad[keep].isnan()) and (y[keep & bad.isinf()] == -math.inf).all()
    assert not torch.equal(ops.dropout(x, 0.5, 7), ops.dropout(x, 0.5, 8))
    assert torch.equal(ops.dropout(x, 0.5, (1 << 64) - 1) == 0, ~philox_keep((1 << 64) - 1, 1000, 0.5) | (x == 0))


@pytest.mark.parametrize("dtype", DTYPES)
def test_dropout_strides(guards, dtype):
    """the mask goes by the element's place in the tensor, whatever its strides; an unaligned start"""
    x = randn((33, 50), 35, dtype)
    want = ops.dropout(x, 0.4, 9)
    assert torch.equal(ops.dropout(x.t().contiguous().t(), 0.4, 9), want)
    wide = randn((1700,), 36, dtype)
    wide[1:1651] = x.reshape(-1)
    assert torch.equal(ops.dropout(wide[1:1651].view(33, 50), 0.4, 9), want)
    leaf = x.clone().requires_grad_()
    (g,) = torch.autograd.grad(ops.dropout(leaf, 0.4, 9).sum(), leaf)       # a broadcast gradient
    assert torch.equal(g == 0, want == 0)
    assert guards.broken_guards() == 0


def test_dropout_large_counters():
    """past 2^32 elements the counter's high word counts: the mask of the tail, by its own counters"""
    n = (1 << 32) + 37
    x = torch.ones((n,), dtype=torch.bfloat16, device=DEV)
    y = ops.dropout(x, 0.5, 10)
    at = n - 1029 - (n - 1029) % 4
    m = np.uint64(0xFFFFFFFF)
    ctr = np.arange(at // 4, (n + 3) // 4, dtype=np.uint64)
    c, k = [ctr & m, ctr >> np.uint64(32), np.zeros_like(ctr), np.zeros_like(ctr)], [10, 0]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & m, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & m]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    w = np.stack(c, -1).reshape(-1)[:n - at]
    keep = torch.from_numpy(((w >> np.uint64(8)).astype(np.float64) + 1.0) * 2.0 ** -24 > 0.5).to(DEV)
    assert torch.equal(y[at:] != 0, keep)
    assert torch.equal(y[:1000] != 0, philox_keep(10, 1000, 0.5))


# ---------------------------------------------------------------------------------------------- rotary positions
def rot_reference(x, pos, freqs, sections, interleaved, sign=1.0):
    out, x, at, f = x.double().clone(), x.double(), 0, 0
    for a, n in enumerate(sections):
        ang = pos[..., a].double()[..., None] * freqs[f:f + n // 2].to(x.device)
        c, s = ang.cos()[..., None, :], sign * ang.sin()[..., None, :]
        first = slice(at, at + n, 2) if interleaved else slice(at, at + n // 2)
        second = slice(at + 1, at + n, 2) if interleaved else slice(at + n // 2, at + n)
        out[..., first] = x[..., first] * c - x[..., second] * s
        out[..., second] = x[..., second] * c + x[..., first] * s
        at, f = at + n, f + n // 2
    return out


def rot_close(got, x, pos, freqs, sections, interleaved, sign=1.0, what=""):
    want = rot_reference(x, pos, freqs, sections, interleaved, sign)
    # sine and cosine on [-pi/4, pi/4] are off by 1.5 steps at most (3 u of a value up to 1), each product and the sum by one half
    # step; the pair's length bounds both products
    length = x.double().abs() * 0
    at = 0
    for n in sections:
        v = x.double()[..., at:at + n]
        a, b = (v[..., 0::2], v[..., 1::2]) if interleaved else (v[..., :n // 2], v[..., n // 2:])
        r = a.abs() + b.abs()
        length[..., at:at + n] = torch.stack([r, r], -1).flatten(-2) if interleaved else torch.cat([r, r], -1)
        at += n
    close(got, want, HALF[x.dtype] * want.abs() + 5 * U * length, what)
    assert torch.equal(got[..., at:], x[..., at:]), what + ": the rest of the head passes through"


ROT_CASES = [  # B, T, H, Hk, D, sections
    (1, 1, 1, 1, 2, (2,)), (2, 3, 1, 1, 8, (4, 4)), (1, 7, 2, 1, 64, (32, 32)), (2, 5, 3, 3, 72, (24, 24, 24)), (1, 9, 6, 2, 80, (16, 24, 24)),
    (2, 4, 2, 1, 40, (10, 14)), (1, 6, 5, 0, 33, (6, 2, 4, 2)), (3, 2, 1, 4, 130, (128,)), (1, 1, 4, 4, 64, (2, 2, 2, 2, 2, 2, 2, 2)),
    (1, 515, 4, 4, 64, (32, 32)), (2, 3, 17, 5, 7, (6,)), (1, 3, 2, 2, 512, (256, 128, 64))]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("case", ROT_CASES)
def test_rotary_sizes(guards, dtype, interleaved, case):
    B, T, H, Hk, D, sections = case
    q = randn((B, T, H, D), 40, dtype).requires_grad_()
    k = randn((B, T, Hk, D), 41, dtype).requires_grad_() if Hk else None
    freqs = ops.rotary_freqs(sections, device=DEV)
    A = len(sections)
    for pos in (torch.randint(-40, 40, (T, A), generator=gen(42), device=DEV, dtype=torch.int32),
                torch.randint(0, 5000, (B, T, A), generator=gen(43), device=DEV), torch.randn((B, T, A), generator=gen(44), device=DEV) * 30):
        yq, yk = ops.rotary(q, k, pos, freqs, sections, interleaved=interleaved)
        dq, dk = randn((B, T, H, D), 45, dtype), randn((B, T, Hk, D), 46, dtype)
        rot_close(yq.detach(), q.detach(), pos, freqs, sections, interleaved, what="q")
        if Hk:
            rot_close(yk.detach(), k.detach(), pos, freqs, sections, interleaved, what="k")
            gq, gk = torch.autograd.grad([yq, yk], [q, k], [dq, dk])
            rot_close(gk, dk, pos, freqs, sections, interleaved, -1.0, "dk")
        else:
            assert yk is None
            (gq,) = torch.autograd.grad(yq, q, dq)
        rot_close(gq, dq, pos, freqs, sections, interleaved, -1.0, "dq")
    assert guards.broken_guards() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T", [(1, 20011), (2, 9001), (5, 1501), (7, 4099), (3000, 3)])
def test_rotary_many_tokens(guards, dtype, B, T):
    """several tokens a workgroup, of several samples where these share their positions, and parts of both at the ends"""
    q, k = randn((B, T, 2, 18), 54, dtype), randn((B, T, 1, 18), 55, dtype)
    freqs = ops.rotary_freqs((8, 6), device=DEV)
    for pos in (torch.randint(0, 300, (T, 2), generator=gen(56), device=DEV), torch.randint(0, 300, (B, T, 2), generator=gen(57), device=DEV)):
        for interleaved in (False, True):
            yq, yk = ops.rotary(q, k, pos, freqs, (8, 6), interleaved)
            rot_close(yq, q, pos, freqs, (8, 6), interleaved, what="q")
            rot_close(yk, k, pos, freqs, (8, 6), interleaved, what="k")
    assert guards.broken_guards() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("how", ["fused product", "odd offset", "heads first", "columns not contiguous"])
def test_rotary_strides(guards, dtype, how):
    B, T, H, Hk, D, sections = 2, 6, 4, 2, 48, (16, 24)
    freqs, pos = ops.rotary_freqs(sections, device=DEV), torch.randint(0, 64, (T, 2), generator=gen(47), device=DEV, dtype=torch.int32)
    if how in ("fused product", "odd offset"):
        o = 0 if how == "fused product" else 5
        qkv = randn((B, T, (H + 2 * Hk) * D + 7), 48, dtype)
        q, k = qkv[..., o:o + H * D].unflatten(-1, (H, D)), qkv[..., o + H * D:o + (H + Hk) * D].unflatten(-1, (Hk, D))
    elif how == "heads first":
        q, k = randn((B, H, T, D), 49, dtype).transpose(1, 2), randn((B, Hk, T, D), 50, dtype).transpose(1, 2)
    else:
        q, k = randn((B, T, D, H), 51, dtype).transpose(2, 3), randn((B, T, D, Hk), 52, dtype).transpose(2, 3)
    yq, yk = ops.rotary(q, k, pos, freqs, sections)
    rot_close(yq, q, pos, freqs, sections, False, what="q")
    rot_close(yk, k, pos, freqs, sections, False, what="k")
    assert guards.broken_guards() == 0


def test_rotary_far_positions():
    """positions of 2^30: a fp32 angle would be off by whole turns"""
    pos = torch.tensor([[1 << 30], [(1 << 30) + 1], [-(1 << 30) - 7], [0]], device=DEV)
    freqs = ops.rotary_freqs((32,), device=DEV)
    q = randn((1, 4, 2, 32), 53)
    yq, _ = ops.rotary(q, None, pos, freqs, (32,))
    want = rot_reference(q, pos, freqs, (32,), False)
    # the 64-bit angle itself: 2^30 times 2^-52 of its steps on either side
    close(yq, want, 12 * U * 5 + 2.0 ** -20, "q")


def test_rotary_is_linear_and_keeps_lengths():
    """the gradient is the transpose: <R q, w> = <q, R' w>, and differences of a linear map are the map"""
    sections, freqs = (8, 8), ops.rotary_freqs((8, 8), device=DEV)
    pos = torch.randint(0, 100, (10, 2), generator=gen(54), device=DEV)
    q, w, d = (randn((2, 10, 3, 20), 55 + i) for i in range(3))
    leaf = q.clone().requires_grad_()
    y, _ = ops.rotary(leaf, None, pos, freqs, sections)
    (g,) = torch.autograd.grad(y, leaf, w)
    lhs, rhs = float((y.double() * w.double()).sum()), float((q.double() * g.double()).sum())
    # 1200 products of size below 30, each off by 10 u of it
    assert abs(lhs - rhs) < 1200 * 30 * 10 * U
    up, down = (ops.rotary(q + s * d, None, pos, freqs, sections)[0].double() for s in (0.5, -0.5))
    assert abs(float(((up - down) * w.double()).sum()) - float((g.double() * d.double()).sum())) < 1200 * 30 * 20 * U
    assert ((y.detach().double().norm(dim=-1) - q.double().norm(dim=-1)).abs() < 20 * 10 * U).all()


def test_rotary_only_one_gradient_wanted():
    freqs, pos = ops.rotary_freqs((8,), device=DEV), torch.arange(4, device=DEV)[:, None]
    q, k = randn((1, 4, 2, 8), 58).requires_grad_(), randn((1, 4, 1, 8), 59).requires_grad_()
    yq, yk = ops.rotary(q, k, pos, freqs, (8,))
    (gk,) = torch.autograd.grad(yk.sum(), k, retain_graph=True)
    rot_close(gk, torch.ones_like(gk), pos, freqs, (8,), False, -1.0, "dk")
    (gq,) = torch.autograd.grad(yq.sum(), q)
    rot_close(gq, torch.ones_like(gq), pos, freqs, (8,), False, -1.0, "dq")


def test_rotary_offsets_past_32_bits():
    T, H, D = 70_003, 250, 128
    q = torch.zeros((1, T, H, D), dtype=torch.bfloat16, device=DEV)
    q[:, -5:] = randn((1, 5, H, D), 92, torch.bfloat16)
    freqs, pos = ops.rotary_freqs((64, 32), device=DEV), torch.randint(0, 300, (T, 2), generator=gen(93), device=DEV)
    y, _ = ops.rotary(q, None, pos, freqs, (64, 32))
    alone, _ = ops.rotary(q[:, -5:].clone(), None, pos[-5:], freqs, (64, 32))
    assert torch.equal(y[:, -5:], alone) and (y[:, :-5:1009] == 0).all()


def test_rotary_empty():
    freqs = ops.rotary_freqs((8,), device=DEV)
    for B, T, H in ((0, 3, 2), (2, 0, 2), (2, 3, 0)):
        y, _ = ops.rotary(torch.zeros((B, T, H, 8), device=DEV), None, torch.zeros((T, 1), dtype=torch.int32, device=DEV), freqs, (8,))
        assert y.shape == (B, T, H, 8)


# ---------------------------------------------------------------------------------------------- streams, graphs, second derivatives
def _chain(x, gamma, beta, pos, freqs, seed):
    y = ops.layer_norm(x, gamma, beta)
    q, _ = ops.rotary(y.view(2, 9, 4, 24), None, pos, freqs, (8, 12))
    return ops.dropout(q.reshape(x.shape), 0.2, seed, res=x)


def test_other_streams_and_concurrent_calls():
    """the same work on two streams at once and on the default one: the same bits (nothing is shared between calls)"""
    x, gamma, beta = randn((18, 96), 60), randn((96,), 61), randn((96,), 62)
    pos, freqs = torch.randint(0, 9, (9, 2), generator=gen(63), device=DEV), ops.rotary_freqs((8, 12), device=DEV)
    leaves = [v.clone().requires_grad_() for v in (x, gamma, beta)]
    dy = randn((18, 96), 64)
    want = torch.autograd.grad(_chain(*leaves, pos, freqs, 3), leaves, dy)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [None, None]
    for rep in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = torch.autograd.grad(_chain(*leaves, pos, freqs, 3), leaves, dy)
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))


def test_captured_graphs_replay():
    """forward and backward captured twice into graphs of their own; every replay of either, with eager work in between, gives the
    eager result of the inputs that are there at that time; the dropout seed follows hip.SEED_DEV"""
    pos, freqs = torch.randint(0, 9, (9, 2), generator=gen(65), device=DEV), ops.rotary_freqs((8, 12), device=DEV)
    dy, offset = randn((18, 96), 66), torch.zeros((1,), dtype=torch.int64, device=DEV)
    sx, gamma, beta = randn((18, 96), 67), randn((96,), 68), randn((96,), 69)
    graphs = []
    hip.SEED_DEV[0] = offset
    try:
        for i in range(2):
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                leaves = [v.detach().requires_grad_() for v in (sx, gamma, beta)]
                torch.autograd.grad(_chain(*leaves, pos, freqs, 100 + i), leaves, dy)
            torch.cuda.current_stream().wait_stream(side)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                leaves = [v.detach().requires_grad_() for v in (sx, gamma, beta)]
                y = _chain(*leaves, pos, freqs, 100 + i)
                out = [y.detach(), *torch.autograd.grad(y, leaves, dy)]
            graphs.append((g, out))
    finally:
        hip.SEED_DEV[0] = None
    for rep in range(3):
        sx.copy_(randn((18, 96), 70 + rep))
        offset.fill_(1000 * rep)
        for i in (0, 1):
            leaves = [v.clone().requires_grad_() for v in (sx, gamma, beta)]
            y = _chain(*leaves, pos, freqs, 100 + i + 1000 * rep)
            want = [y.detach(), *torch.autograd.grad(y, leaves, dy)]
            graphs[i][0].replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(graphs[i][1], want)), (rep, i)


def test_second_derivatives_are_refused():
    x = randn((4, 16), 80).requires_grad_()
    for y in (ops.layer_norm(x), ops.dropout(x, 0.5, 1)):
        (g,) = torch.autograd.grad(y.square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError):
            g.sum().backward()

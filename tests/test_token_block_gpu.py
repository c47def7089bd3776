"""The token operators together, as a block over image tokens uses them: pre-norm attention with rotary positions over height and width and
a window with sinks, the residual branch through dropout, a second norm and an MLP -- on the library's own linear layers (fp32) or torch's
matrix products (bf16) -- against the same block in 64 bits, forward and every gradient; then a few optimisation steps of it, eager and
from a captured graph."""
import math

import numpy as np
import pytest
import torch

from indm_amd import hip, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U, HALF16 = 2.0 ** -24, 2.0 ** -8
B, HW, H, HK, D, C = 2, 12, 4, 2, 24, 96      # 144 tokens
SECTIONS, WINDOW, SINKS, P, SEED = (8, 12), 30, 2, 0.2, 1234


def keep_mask(seed, n, p):
    m = np.uint64(0xFFFFFFFF)
    c = [np.arange((n + 3) // 4, dtype=np.uint64)] + [np.zeros((n + 3) // 4, dtype=np.uint64) for _ in range(3)]
    k = [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & m, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & m]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    w = np.stack(c, -1).reshape(-1)[:n]
    return torch.from_numpy(((w >> np.uint64(8)).astype(np.float64) + 1.0) * 2.0 ** -24 > float(np.float32(p))).to(DEV)


def weights(dtype):
    g = torch.Generator(device=DEV).manual_seed(1)
    r = lambda *s, sc=1.0: torch.randn(s, generator=g, device=DEV) * sc  # noqa: E731
    w = dict(g1=1 + r(C, sc=0.1), b1=r(C, sc=0.1), g2=1 + r(C, sc=0.1), b2=r(C, sc=0.1), qkv=r((H + 2 * HK) * D, C, sc=C ** -0.5).to(dtype),
             out=r(C, H * D, sc=(H * D) ** -0.5).to(dtype), up=r(2 * C, C, sc=C ** -0.5).to(dtype), down=r(C, 2 * C, sc=(2 * C) ** -0.5).to(dtype))
    return w, r(B, HW * HW, C).to(dtype), r(B, HW * HW, C).to(dtype)


def positions():
    ij = torch.arange(HW, device=DEV)
    return torch.stack(torch.meshgrid(ij, ij, indexing="ij"), -1).view(-1, 2).to(torch.int32)


def block(x, w, pos, freqs, lengths, seed):
    linear = ops.linear if x.dtype == torch.float32 else torch.nn.functional.linear
    y = ops.layer_norm(x, w["g1"], w["b1"])
    qkv = linear(y, w["qkv"])
    q, k, v = (t.unflatten(-1, (-1, D)) for t in qkv.split([H * D, HK * D, HK * D], -1))
    q, k = ops.rotary(q, k, pos, freqs, SECTIONS)
    o = ops.window_attention(q, k, v, WINDOW, sinks=SINKS, lengths=lengths)
    x = ops.dropout(linear(o.flatten(-2), w["out"]), P, seed, res=x)
    y = ops.layer_norm(x, w["g2"], w["b2"])
    return ops.dropout(linear(torch.relu(linear(y, w["up"])), w["down"]), P, seed + 1, res=x)


def block64(x, w, pos, freqs, lengths, seed):
    """the definition, in x's (64-bit) type"""
    def norm(x, g, b):
        d = x - x.mean(-1, keepdim=True)
        return d / torch.sqrt((d * d).mean(-1, keepdim=True) + 1e-6) * g + b

    def turn(t):
        at, f, parts = 0, 0, []
        for a, n in enumerate(SECTIONS):
            ang = (pos[:, a].double()[:, None] * freqs[f:f + n // 2])[:, None]
            p, m = t[..., at:at + n // 2], t[..., at + n // 2:at + n]
            parts += [p * ang.cos() - m * ang.sin(), m * ang.cos() + p * ang.sin()]
            at, f = at + n, f + n // 2
        return torch.cat(parts + [t[..., at:]], -1)

    def drop(t, s, res):
        return res + t * keep_mask(s, t.numel(), P).view_as(t) / (1 - float(np.float32(P)))

    T = x.shape[1]
    y = norm(x, w["g1"], w["b1"]) @ w["qkv"].t()
    q, k, v = (t.unflatten(-1, (-1, D)) for t in y.split([H * D, HK * D, HK * D], -1))
    q, k = turn(q).transpose(1, 2), turn(k).transpose(1, 2).repeat_interleave(H // HK, 1)
    v = v.transpose(1, 2).repeat_interleave(H // HK, 1)
    i, j = torch.arange(T, device=DEV)[:, None], torch.arange(T, device=DEV)[None]
    see = (((i - j).abs() <= WINDOW) | (j < SINKS))[None] & (i < lengths[:, None, None]) & (j < lengths[:, None, None])
    z = (q @ k.transpose(-1, -2) * D ** -0.5).masked_fill(~see[:, None], -math.inf)
    top = z.amax(-1, keepdim=True).detach()
    e = torch.exp(z - torch.where(top == -math.inf, 0.0, top))
    s = e.sum(-1, keepdim=True)
    o = (e / torch.where(s == 0, 1.0, s)) @ v
    x = drop(o.transpose(1, 2).flatten(-2) @ w["out"].t(), seed, x)
    return drop(torch.relu(norm(x, w["g2"], w["b2"]) @ w["up"].t()) @ w["down"].t(), seed + 1, x)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_block_forward_and_gradients(dtype):
    """The 2-norm of each result's error against the 2-norm of the result.  fp32: 11 operators, each off by a few u of its 96- to 192-term
    sums (at most 200 u), forward, and twice as many backward: 11 x 200 u x 3 = 4e-4 bounds it without any averaging.  bf16: each
    operator rounds its result (h / 2 in the mean square, less than h), the rounded values of 11 forward and 22 backward steps meet in
    a gradient: sqrt(33) h = 2.3e-2 if they are independent, all in one direction 33 h; twice the former.

    The relu adds to that, for what lies before it: its inputs a are near N(0, 1) (normalised rows times weights of variance 1 / C), off by
    d of at most sqrt(8) h = 0.011 in the mean square after eight rounded results.  A sign differs with probability density(0) E|d| =
    0.4 x 0.8 x 0.011 = 0.0035, and there the whole gradient of the entry comes or goes; half of the entries pass one, so the relative
    square of the error is 0.0035 / 0.5 = 0.007, its root 0.084.  (In fp32 the inputs are off by some u, 55296 of them: 0.02 flips expected.)"""
    w, x, dy = weights(dtype)
    pos, freqs = positions(), ops.rotary_freqs(SECTIONS, device=DEV)
    lengths = torch.tensor([HW * HW, 100], dtype=torch.int32, device=DEV)
    names = sorted(w)
    leaves = [x.clone().requires_grad_()] + [w[n].clone().requires_grad_() for n in names]
    y = block(leaves[0], dict(zip(names, leaves[1:])), pos, freqs, lengths, SEED)
    got = [y, *torch.autograd.grad(y, leaves, dy)]
    wide = [t.detach().double().requires_grad_() for t in leaves]
    y64 = block64(wide[0], dict(zip(names, wide[1:])), pos, freqs, lengths, SEED)
    want = [y64, *torch.autograd.grad(y64, wide, dy.double())]
    for name, a, b in zip(["y", "dx"] + names, got, want):
        rel = float((a.detach().double() - b.detach()).norm() / b.detach().norm())
        bound = 4e-4 if dtype == torch.float32 else 2 * math.sqrt(33) * HALF16 + (0.0 if name in ("y", "down") else 0.084)
        assert rel < bound, (name, rel)


def test_block_trains_the_same_from_a_captured_graph():
    """four steps of plain gradient descent with another dropout seed each: eager, and one captured forward + backward that is replayed with
    the seed's offset in device memory -- the same bits in every weight after every step"""
    dtype = torch.bfloat16
    pos, freqs = positions(), ops.rotary_freqs(SECTIONS, device=DEV)
    lengths = torch.tensor([HW * HW, 77], dtype=torch.int32, device=DEV)
    names = sorted(weights(dtype)[0])

    def grads(w, x, dy, seed):
        leaves = [w[n].detach().requires_grad_() for n in names]
        y = block(x, dict(zip(names, leaves)), pos, freqs, lengths, seed)
        return torch.autograd.grad(y, leaves, dy)

    def descend(w, g):
        for n, d in zip(names, g):
            w[n].sub_((d.float() * 1e-3).to(w[n].dtype))

    w, x, dy = weights(dtype)
    eager = []
    for step in range(4):
        descend(w, grads(w, x, dy, SEED + 10 * step))
        eager.append([w[n].clone() for n in names])

    w, x, dy = weights(dtype)
    offset = torch.zeros((1,), dtype=torch.int64, device=DEV)
    hip.SEED_DEV[0] = offset
    try:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            grads(w, x, dy, SEED)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            g = grads(w, x, dy, SEED)
    finally:
        hip.SEED_DEV[0] = None
    for step in range(4):
        offset.fill_(10 * step)
        graph.replay()
        descend(w, g)
        torch.cuda.synchronize()
        for n, a, b in zip(names, eager[step], (w[n] for n in names)):
            assert torch.equal(a, b), (step, n)

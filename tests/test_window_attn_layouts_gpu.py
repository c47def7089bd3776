"""Every compiled layout of the window attention kernels -- wavefronts that share a block of queries or keys or own one each, key blocks whose
queries are split, the sinks' workgroups behind the key blocks' or in a launch of their own -- at every padded head width, in both types, with
sinks, sequences that end among them and an empty one, against 64 bits (window_attn_bounds.py) with guard bands."""
import math

import pytest
import torch

from indm_amd import hip, ops
from window_attn_bounds import close, definition

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture
def guards():
    ext = hip.token_ops()
    ext.guard(1 << 16)
    try:
        yield ext
    finally:
        ext.broken_guards()
        ext.guard(0)


def layout(dtype, B, T, H, Hk, D, left, right, sinks, causal):
    r = hip.lib().indm_wattn_layout(2 if dtype == torch.bfloat16 else 4, B, T, H, Hk, D, left, right, sinks, int(causal))
    assert r >= 0
    return dict(queries=bool(r & 1), keys=bool(r & 2), apart=bool(r & 4), split=(r >> 4 & 0xfff) > 1, sinks=r >> 16 > 0)


def randn(shape, seed, dtype, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV) * scale).to(dtype)


def run(q, k, v, do, left, right, sinks, causal, lengths=None):
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    o = ops.window_attention(*leaves, (left, right), sinks=sinks, causal=causal, lengths=lengths)
    return [o.detach(), *torch.autograd.grad(o, leaves, do)]


def check(q, k, v, do, left, right, sinks, causal, lengths=None):
    got, xs = run(q, k, v, do, left, right, sinks, causal, lengths), (q, k, v, do)
    if lengths is not None:
        dead = torch.arange(q.shape[1], device=DEV)[None, :] >= lengths.clamp(0, q.shape[1])[:, None]
        xs = [x.masked_fill(dead[:, :, None, None], 0.0) for x in xs]
    want, err = definition(*xs, left, right, sinks, causal, lengths)
    for name, a, w, e in zip(("o", "dq", "dk", "dv"), got, want, err):
        close(a, w, e, name)
        assert lengths is None or (a[dead] == 0).all(), name
    return got


#  what the layout has to be (the sinks aside): queries shared, keys shared, queries of a key block split;  B, T, H, Hk, left, right, sinks
LAYOUTS = {
    "own blocks": ((False, False, False), (40, 300, 4, 4, 30, 20, 5)),
    "own blocks, many sinks": ((False, False, False), (40, 300, 4, 4, 9, 4, 150)),
    "split": ((False, False, True), (5, 600, 8, 2, 300, 100, 16)),
    "split, no sinks": ((False, False, True), (5, 600, 8, 2, 300, 100, 0)),
    "shared": ((True, True, False), (3, 260, 4, 4, 20, 30, 5)),
    "shared and split": ((True, True, True), (1, 500, 8, 2, 260, 200, 40)),
    "own blocks, no sinks": ((False, False, False), (40, 300, 4, 4, 30, 20, 0)),
    "own queries, shared keys": ((False, True, True), (3, 700, 8, 1, 20, 8, 3)),
}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("D", [32, 40, 64, 72, 96, 128])
@pytest.mark.parametrize("name", LAYOUTS)
def test_layouts(guards, dtype, causal, D, name):
    (queries, keys, split), (B, T, H, Hk, left, right, sinks) = LAYOUTS[name]
    got = layout(dtype, B, T, H, Hk, D, left, right, sinks, causal)
    assert got == dict(queries=queries, keys=keys, split=split, sinks=sinks > 0, apart=sinks > 0 and not keys and not split), got
    q, k, v, do = (randn((B, T, h, D), 1 + i, dtype, 1.3 if i < 2 else 1.0) for i, h in enumerate((H, Hk, Hk, H)))
    n = [T, T - 1, sinks // 2, 0, 129, T, 33]
    lengths = torch.tensor([n[b % len(n)] for b in range(B)], dtype=torch.int32, device=DEV)
    dead = torch.arange(T, device=DEV)[None, :] >= lengths[:, None]
    for x, bad in zip((q, k, v, do), (math.nan, math.inf, -math.inf, math.nan)):
        x[dead] = bad       # what lies behind a sequence is nobody's
    got = check(q, k, v, do, left, right, sinks, causal, lengths)
    assert guards.broken_guards() == 0
    assert all(torch.equal(a, b) for a, b in zip(got, run(q, k, v, do, left, right, sinks, causal, lengths)))     # the same bits again


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("B,T,H,Hk,D", [(1, 2048, 2, 1, 64), (2, 1031, 4, 4, 32), (1, 4096, 1, 1, 128)])
def test_every_token_sees_every_other(guards, dtype, causal, B, T, H, Hk, D):
    """the default call, window=None, past a thousand tokens"""
    q, k, v, do = (randn((B, T, h, D), 11 + i, dtype) for i, h in enumerate((H, Hk, Hk, H)))
    got = check(q, k, v, do, T, T, 0, causal)
    with torch.no_grad():
        assert torch.equal(ops.window_attention(q, k, v, causal=causal), got[0])
    assert guards.broken_guards() == 0

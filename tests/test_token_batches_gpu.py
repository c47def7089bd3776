"""Layer norm and rotary positions at the sizes where a team takes several rows at once and a workgroup several samples, and the operators'
measured cases (perf/operators.py) against their definition in 64 bits."""
import importlib.util
import os

import pytest
import torch

import test_token_ops_gpu as base
from indm_amd import hip, ops
from window_attn_bounds import one_rounding

pytestmark = pytest.mark.gpu
DEV, U = base.DEV, base.U
DTYPES = [torch.float32, torch.bfloat16]
guards = base.guards


# Rows just past the numbers from which a team takes two or four at once (forward 512 x teams x rows, backward workgroups x teams x rows), with a
# remainder: teams of 16, 32 and 64 lanes with one to four vectors.
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,C", [(32771, 48), (16389, 100), (16389, 256), (8195, 320), (8195, 511), (4099, 700), (4099, 1000)])
def test_layer_norm_several_rows_a_team(guards, dtype, R, C):
    x = base.randn((R, C), 1, dtype, 2.0, 0.4).requires_grad_()
    gamma, beta = base.randn((C,), 2, scale=0.3, mean=1.0).requires_grad_(), base.randn((C,), 3).requires_grad_()
    dy = base.randn((R, C), 4, dtype)
    y = ops.layer_norm(x, gamma, beta)
    dx, dg, db = torch.autograd.grad(y, (x, gamma, beta), dy)
    base.ln_check(x.detach(), gamma.detach(), beta.detach(), 1e-6, dy, y.detach(), dx, None, None)
    # the columns' sums: a team adds at most 9 rows one after another (256 workgroups or more), 16 teams, 32 runs of at most 32 workgroups, and 5
    # steps across the runs: 64 + 32 additions; and each term's own error, three products of fp32 values on top of xh's
    xd, dyd = x.detach().double(), dy.double()
    m = xd.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt(((xd - m) ** 2).mean(1, keepdim=True) + 1e-6)
    xh = (xd - m) * rstd
    err_xh = U * (50 * xd.abs().amax(1, keepdim=True) * rstd + 52 * xh.abs())
    base.close(dg, (dyd * xh).sum(0), (U * 99 * (dyd * xh).abs() + err_xh * dyd.abs()).sum(0), "dgamma")
    base.close(db, dyd.sum(0), (U * 99 * dyd.abs()).sum(0), "dbeta")
    with torch.no_grad():
        assert torch.equal(ops.layer_norm(x, gamma, beta), y)
    # a row's result does not depend on how many rows there are
    few = slice(R - 40, R)
    part = x.detach()[few].clone().requires_grad_()
    yp = ops.layer_norm(part, gamma, beta)
    assert torch.equal(yp, y[few]) and torch.equal(torch.autograd.grad(yp, part, dy[few])[0], dx[few])
    assert guards.broken_guards() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,T,H,Hk,D,sections", [(5, 2003, 4, 4, 64, (32, 32)), (7, 1801, 8, 2, 64, (32, 32)), (2, 4001, 2, 1, 80, (16, 24, 24)),
                                                 (64, 257, 4, 4, 64, (32, 32)), (6, 1024, 2, 2, 256, (128, 128))])
def test_rotary_samples_that_share_positions(guards, dtype, interleaved, B, T, H, Hk, D, sections):
    """whole vectors with their mates, several samples a workgroup, forward and backward, out of one fused product"""
    qkv = base.randn((B, T, (H + 2 * Hk) * D), 5, dtype)
    q, k = (t.requires_grad_() for t in (qkv[..., :H * D].unflatten(-1, (H, D)), qkv[..., H * D:(H + Hk) * D].unflatten(-1, (Hk, D))))
    freqs = ops.rotary_freqs(sections, device=DEV)
    pos = torch.randint(0, 300, (T, len(sections)), generator=base.gen(6), device=DEV, dtype=torch.int32)
    dq, dk = base.randn((B, T, H, D), 7, dtype), base.randn((B, T, Hk, D), 8, dtype)
    yq, yk = ops.rotary(q, k, pos, freqs, sections, interleaved)
    gq, gk = torch.autograd.grad([yq, yk], [q, k], [dq, dk])
    for got, x, sign, what in ((yq, q, 1.0, "q"), (yk, k, 1.0, "k"), (gq, dq, -1.0, "dq"), (gk, dk, -1.0, "dk")):
        base.rot_close(got.detach(), x.detach(), pos, freqs, sections, interleaved, sign, what)
    assert guards.broken_guards() == 0


def cases():
    spec = importlib.util.spec_from_file_location("operator_cases", os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "perf", "operators.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("name", [c["name"] for c in cases().listed()])
def test_measured_cases(guards, name):
    """The 2-norm of the error of every output.  bfloat16: one rounding's.  float32: a value gathers up to 4096 roundings of random sign
    (attention's sums over a sequence, the columns' sums), each half a step u of its terms at most, u / sqrt(3) in the mean square: 64 / sqrt(3) = 37 u
    of the norm, where terms of one sign do not cancel; twice that where they do."""
    module = cases()
    case = next(c for c in module.listed() if c["name"] == name)
    module.own = True
    got = module.run(module.prepare(case, 11))
    want = module.exact(case, 11)
    assert len(got) == len(want)
    for i, (a, w) in enumerate(zip(got, want)):
        a = a.detach()
        assert a.shape == w.shape and a.isfinite().all()
        if a.dtype == torch.bfloat16:
            one_rounding(a, w, f"{name} output {i}")
        else:
            assert float((a.double() - w).norm()) <= 74 * U * float(w.norm()), (name, i)
    assert guards.broken_guards() == 0

"""Window attention holds what one rounding of the exact result holds: bounds without a rounding of any operand (window_attn_bounds.py;
test_window_attn_precision_cpu.py shows what they catch), in both types, forward and gradients."""
import pytest
import torch

from indm_amd import ops
from window_attn_bounds import close, definition, one_rounding

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset", [0.0, 8.0])     # 8: the values' common part, which dP - <dO, o> has to cancel
@pytest.mark.parametrize("B,T,H,Hk,D,left,right,sinks,causal", [
    (1, 200, 1, 1, 64, 30, 30, 2, False), (2, 333, 4, 2, 40, 60, 0, 5, True), (1, 130, 2, 1, 128, 130, 130, 0, False), (3, 257, 2, 2, 24, 9, 31, 3, False),
    (40, 300, 4, 4, 64, 30, 20, 5, False), (5, 600, 8, 2, 128, 300, 0, 16, True), (4, 520, 8, 4, 96, 100, 100, 0, False)])
def test_one_rounding(dtype, offset, B, T, H, Hk, D, left, right, sinks, causal):
    g = torch.Generator(device=DEV).manual_seed(7)
    q, k, v, do = ((torch.randn((B, T, h, D), generator=g, device=DEV) * s + a).to(dtype)
                   for h, s, a in ((H, 1.3, 0), (Hk, 1.3, 0), (Hk, 1, offset), (H, 1, 0)))
    leaves = [x.requires_grad_() for x in (q, k, v)]
    o = ops.window_attention(*leaves, (left, right), sinks=sinks, causal=causal)
    got = [o.detach(), *torch.autograd.grad(o, leaves, do)]
    want, err = definition(*(x.detach() for x in (q, k, v)), do, left, right, sinks, causal)
    for name, a, w, e in zip(("o", "dq", "dk", "dv"), got, want, err):
        close(a, w, e, name)
        if dtype == torch.bfloat16:
            one_rounding(a, w, name)

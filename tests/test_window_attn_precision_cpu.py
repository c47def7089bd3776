"""The bounds of window_attn_bounds.py against an emulation of the kernels' operand roundings: as the kernels work it passes, and each
single loss of a digit -- an operand without its rest, a wrong rest of o -- fails."""
import pytest
import torch

from window_attn_bounds import close, definition, one_rounding, visible

BF16 = torch.bfloat16


def rounded(x):
    return x.to(BF16).double()


def two(x):
    return rounded(x) + rounded(x - rounded(x))


def emulated(q, k, v, do, left, right, sinks, causal, lost=None):
    """o, dq, dk, dv of one head with its operands rounded as the kernels round them; lost: which digits go missing"""
    T, D = q.shape[1], q.shape[3]
    Q, K, V, dO = (x[0, :, 0].double() for x in (q, k, v, do))
    see = visible(T, left, right, sinks, causal, T)
    P = torch.softmax((Q @ K.t() * D ** -0.5).masked_fill(~see, -torch.inf), 1)
    O = (rounded(P) if lost == "P of o" else two(P)) @ V
    o = O.to(BF16)
    rest = rounded(O - o.double())
    rest = {"rest of o": 0 * rest, "sign of the rest": -rest, "row of the rest": rest.roll(1, 0)}.get(lost, rest)
    dS = P * (dO @ V.t() - (dO * (o.double() + rest)).sum(1, keepdim=True))
    dq = (rounded(dS) if lost == "dS of dq" else two(dS)) @ K * D ** -0.5
    dk = (rounded(dS) if lost == "dS of dk" else two(dS)).t() @ Q * D ** -0.5
    dv = (rounded(P) if lost == "P of dv" else two(P)).t() @ dO
    return [x.to(BF16)[None, :, None] for x in (o, dq, dk, dv)]


def case(offset):
    g = torch.Generator().manual_seed(3)
    q, k, v, do = ((torch.randn((1, 200, 1, 64), generator=g) * s + a).to(BF16) for s, a in ((1.3, 0), (1.3, 0), (1, offset), (1, 0)))
    return (q, k, v, do), (30, 30, 2, False)


def passes(xs, window, lost):
    want, err = definition(*xs, *window)
    try:
        for name, got, w, e in zip(("o", "dq", "dk", "dv"), emulated(*xs, *window, lost), want, err):
            close(got, w, e, name)
            one_rounding(got, w, name)
    except AssertionError:
        return False
    return True


@pytest.mark.parametrize("offset", [0.0, 8.0])
def test_two_operands_pass(offset):
    assert passes(*case(offset), None)


@pytest.mark.parametrize("lost,offset", [("P of o", 0.0), ("dS of dq", 0.0), ("dS of dk", 0.0), ("P of dv", 0.0), ("rest of o", 8.0),
                                         ("sign of the rest", 8.0), ("row of the rest", 8.0)])
def test_lost_digits_fail(lost, offset):
    assert not passes(*case(offset), lost)

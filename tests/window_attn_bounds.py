"""The definition of window attention in 64 bits with bounds that count the kernels' roundings, for results of either type.

u = 2^-24 is half a step of fp32.  What the kernels hold in bf16 as two operands -- P and dS in their second products, o next to what its
rounding left -- is off by 2^-8 of 2^-8 of itself, s = 2^-16; in fp32 the operands are the values, s = 0.  Everything else is fp32:
  logits   z = scale q.k: D products and sums, (D + 4) u scale |q|.|k|; the exponent adds 2 u |z| + 2 u |lse|, exp2 and the row's sum of N
           terms 8 u + N u.  P is off by that relative error, its own and, through the sum, its row's largest: E = 2 max.
  o        sum P v, two operands a term: s + E + (2 N + 4) u of sum P |v|
  delta    <dO, o> from o and its rest: s |o| and o's error, times |dO|, and 2 D sums
  dS       P (dP - delta): E + 4 u of itself, and P times the errors of dP (D products) and of delta
  dq, dk   scale times sums of dS k, dS q: dS' error and s of it, (2 N + 16) u of the sum of the terms' sizes;  dv: sum P dO likewise
These bound the value x before its one rounding to the tensors' type, |x - want| <= e.  The rounding takes the nearest: |round(x) - x| <=
|round(want) - x| <= |round(want) - want| + e, so that |round(x) - want| <= |round(want) - want| + 2 e."""
import math

import torch

U = 2.0 ** -24


def visible(T, left, right, sinks, causal, n, device="cpu"):
    """[T, T]: key j is visible to query i of a sequence of n"""
    i = torch.arange(T, device=device)[:, None]
    j = torch.arange(T, device=device)[None, :]
    m = ((j >= i - left) & (j <= i + right)) | (j < sinks)
    if causal:
        m = m & (j <= i)
    return m & (i < n) & (j < n)


def definition(q, k, v, do, left, right, sinks=0, causal=False, lengths=None, scale=None):
    """-> [o, dq, dk, dv] in 64 bits, and the bounds e of the values before their rounding"""
    B, T, H, D = q.shape
    Hk = k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    s = 2.0 ** -16 if q.dtype == torch.bfloat16 else 0.0
    q64, k64, v64, do64 = (x.double() for x in (q, k, v, do))
    want = [torch.zeros_like(x) for x in (q64, q64, k64, v64)]
    err = [torch.zeros_like(x) for x in (q64, q64, k64, v64)]
    mm = lambda a, c: a @ c.contiguous()  # noqa: E731
    for b in range(B):
        n = T if lengths is None else max(0, min(T, int(lengths[b])))
        if n == 0:
            continue
        see = visible(T, left, right, sinks, causal, n, q.device)[:n, :n]
        N, Nk = int(see.sum(1).max()), int(see.sum(0).max()) * (H // Hk)
        for h in range(H):
            g = h // (H // Hk)
            Q, K, V, dO = (x.contiguous() for x in (q64[b, :n, h], k64[b, :n, g], v64[b, :n, g], do64[b, :n, h]))
            z = mm(Q, K.t()) * scale
            zm = z.masked_fill(~see, -math.inf)
            lse = zm.logsumexp(1, keepdim=True)
            P = torch.exp(zm - lse)
            E = U * ((D + 4) * scale * mm(Q.abs(), K.abs().t()) + 2 * z.abs() + 2 * lse.abs() + 8 + N)
            E = 2 * E.masked_fill(~see, 0.0).amax(1, keepdim=True)
            O = mm(P, V)
            eo = mm(P, V.abs()) * (s + E + (2 * N + 4) * U) + 2 * U * O.abs()
            dP, delta = mm(dO, V.t()), (dO * O).sum(1, keepdim=True)
            edelta = (dO.abs() * (eo + s * O.abs())).sum(1, keepdim=True) + (2 * D + 4) * U * (dO * O).abs().sum(1, keepdim=True)
            dS = P * (dP - delta)
            eS = dS.abs() * (s + E + 4 * U) + P * ((D + 4) * U * mm(dO.abs(), V.abs().t()) + edelta)
            PT, dST, eST = (x.t().contiguous() for x in (P, dS, eS))
            want[0][b, :n, h], err[0][b, :n, h] = O, eo
            want[1][b, :n, h] = scale * mm(dS, K)
            err[1][b, :n, h] = scale * (mm(eS, K.abs()) + (2 * N + 16) * U * mm(dS.abs(), K.abs()))
            want[2][b, :n, g] += scale * mm(dST, Q)
            err[2][b, :n, g] += scale * (mm(eST, Q.abs()) + (2 * Nk + 16) * U * mm(dST.abs(), Q.abs()))
            want[3][b, :n, g] += mm(PT, dO)
            err[3][b, :n, g] += mm((P * (s + E + (2 * Nk + 16) * U)).t().contiguous(), dO.abs())
    return want, err


def close(got, want, err, what=""):
    d, room = (got.double() - want).abs(), (want.to(got.dtype).double() - want).abs() + 2 * err
    bad = ~(d <= room)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}, worst {float((d - room)[bad].max())} over"


def one_rounding(got, want, what=""):
    """The 2-norm of the error is at most 1.02 of that of the exact result's rounding.  Before its rounding a value is off by some d; the
    rounding's own error is spread over a step t, so the mean square is t^2 / 12 + d^2.  The bound holds up to d = 0.2 times the
    rounding's error in the mean square; errors of 2^-16 and of fp32's sums are a twentieth of it at most, a second rounding to the
    type is all of it (1.41)."""
    got, own = (got.double() - want).norm(), (want.to(got.dtype).double() - want).norm()
    assert got <= 1.02 * own, f"{what}: error {float(got / want.norm()):.3g} of the norm, one rounding has {float(own / want.norm()):.3g}"

"""Cases that measure the token operators of indm_amd.ops: layer norm, counter-based dropout, rotary positions over
several axes, and attention over a sliding window with sink tokens.

`listed()` are the cases by name, `draw(rng)` gives more of the same ranges.  `prepare(case, seed)` makes what a program has
in hand before the call, `run(state)` is one pass, `work(case)` what a pass has to move and compute, `exact(case, seed)` the
definition in 64 bits.  With `own` false `run` computes the operators in elementary torch operations."""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "bf16": 2}
EPS = 1e-6          # the eps of the score network's norms
LARGEST = 1 << 25   # elements of the largest tensor of a case (128 images x 32 x 32 tokens x 256 channels)
PAIRS = 1 << 29     # query-key pairs B * H * T * T of the largest attention case (8 images x 4 heads, 64 x 64 tokens)


def listed():
    return [
        # one 32 x 32 image at the attention resolution while sampling: 16 x 16 tokens of 256 channels, latency only
        dict(name="layer_norm_one_image", op="layer_norm", dtype="bf16", train=False, affine=True, sliced=False, rows=256, C=256),
        # a training step's batch of 128 images, 32 x 32 tokens of 256 channels
        dict(name="layer_norm_batch", op="layer_norm", dtype="bf16", train=True, affine=True, sliced=False, rows=131072, C=256),
        # an odd width and row count in single precision, read as a column slice of a wider product
        dict(name="layer_norm_odd", op="layer_norm", dtype="f32", train=True, affine=True, sliced=True, rows=4099, C=1153),
        # the residual branch of a training step's batch: res + dropout(x)
        dict(name="dropout_residual_batch", op="dropout", dtype="bf16", train=True, residual=True, p=0.1, n=LARGEST),
        # the per-rank shard of 16 images in single precision, a size that is no multiple of a vector
        dict(name="dropout_odd", op="dropout", dtype="f32", train=True, residual=False, p=0.1, n=16 * 1024 * 256 + 3),
        # height and width positions of 32 x 32 tokens for the queries and keys of one fused product, a batch of 64
        dict(name="rotary_image_batch", op="rotary", dtype="bf16", train=True, interleaved=False, scaled=False, per_row=False,
             B=64, t=1, h=32, w=32, H=4, Hk=4, D=64, d_t=0, d_h=32, d_w=32),
        # time, height and width of a short clip with odd extents, shared key heads, part of the head left unrotated
        dict(name="rotary_clip_odd", op="rotary", dtype="f32", train=True, interleaved=True, scaled=True, per_row=True,
             B=3, t=7, h=17, w=15, H=6, Hk=2, D=80, d_t=16, d_h=24, d_w=24),
        # one image at the attention resolution while sampling
        dict(name="rotary_one_image", op="rotary", dtype="bf16", train=False, interleaved=False, scaled=False, per_row=False,
             B=1, t=1, h=16, w=16, H=4, Hk=4, D=64, d_t=0, d_h=32, d_w=32),
        # one image at the attention resolution while sampling: 256 tokens, a window of four token rows to each side
        dict(name="attention_one_image", op="attention", dtype="bf16", train=False, ragged=False, causal=False,
             B=1, T=256, H=4, Hk=4, D=64, left=64, right=64, sinks=1),
        # training on 64 x 64 tokens (CelebA at full resolution): a window of four token rows to each side, four sinks
        dict(name="attention_batch", op="attention", dtype="bf16", train=True, ragged=False, causal=False,
             B=8, T=4096, H=4, Hk=4, D=64, left=256, right=256, sinks=4),
        # wide heads that share their keys, in raster order (causal), sequences of different lengths
        dict(name="attention_ragged", op="attention", dtype="bf16", train=True, ragged=True, causal=True,
             B=5, T=1543, H=8, Hk=2, D=128, left=500, right=0, sinks=16),
        # single precision, odd length, a head width that is no power of two
        dict(name="attention_odd", op="attention", dtype="f32", train=True, ragged=False, causal=False,
             B=2, T=1021, H=4, Hk=4, D=40, left=100, right=27, sinks=3),
    ]


def _log_int(rng, low, high):
    """a whole number of [low, high], spread over the logarithm"""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["layer_norm", "dropout", "rotary", "attention"])
    case = dict(op=op, dtype=rng.choice(["f32", "bf16"]), train=rng.random() < 0.7)
    if op == "layer_norm":
        C = _log_int(rng, 16, 8192)
        if rng.random() < 0.5:
            C = max(16, C // 16 * 16)
        rows = _log_int(rng, 1, max(1, min(131072, LARGEST // C)))
        if case["train"]:
            rows = max(rows, 2)
        case.update(affine=rng.random() < 0.8, sliced=rng.random() < 0.3, rows=rows, C=C)
    elif op == "dropout":
        case.update(residual=rng.random() < 0.5, p=rng.choice([0.05, 0.1, 0.1, 0.25, 0.5]), n=_log_int(rng, 256, LARGEST))
    elif op == "rotary":
        t, h, w = rng.choice([1, 1, _log_int(rng, 2, 16)]), _log_int(rng, 1, 64), _log_int(rng, 1, 64)
        d_t = 2 * rng.randint(1, 16) if t > 1 else 0
        d_h, d_w = 2 * rng.randint(2, 16), 2 * rng.randint(2, 16)
        D = (d_t + d_h + d_w + 7) // 8 * 8 + rng.choice([0, 0, 8, 32])
        Hk = rng.choice([1, 2, 3, 4, 8])
        H = Hk * rng.choice([1, 1, 2, 4])
        B = _log_int(rng, 1, max(1, min(64, LARGEST // 2 // (t * h * w * H * D))))
        case.update(interleaved=rng.random() < 0.5, scaled=rng.random() < 0.5, per_row=rng.random() < 0.3, B=B, t=t, h=h, w=w, H=H, Hk=Hk,
                    D=D, d_t=d_t, d_h=d_h, d_w=d_w)
    else:
        D = rng.choice([32, 40, 64, 64, 72, 96, 128])
        Hk = rng.choice([1, 2, 3, 4])
        H = Hk * rng.choice([1, 1, 2, 4])
        # no dearer than the largest listed case, whose windows are half as wide: half its pairs at its head width, in f32 an eighth
        most = PAIRS * 64 // max(64, D) // (2 if case["dtype"] == "bf16" else 8)
        T = _log_int(rng, 2 if case["train"] else 1, min(4096, math.isqrt(most // H)))
        B = _log_int(rng, 1, max(1, min(16, most // (H * T * T))))
        causal = rng.random() < 0.4
        case.update(ragged=rng.random() < 0.4, causal=causal, B=B, T=T, H=H, Hk=Hk, D=D, left=_log_int(rng, 8, 512),
                    right=0 if causal else _log_int(rng, 8, 512), sinks=rng.choice([0, 1, 4, rng.randint(2, 64)]))
    return case


def _normal(gen, shape, dtype, scale=1.0, mean=0.0):
    return (torch.randn(shape, generator=gen, device=gen.device) * scale + mean).to(dtype)


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))
    dtype, train, op = DTYPES[case["dtype"]], case["train"], case["op"]
    s = dict(case=case)
    leaf = lambda t: t.requires_grad_() if train else t  # noqa: E731
    if op == "layer_norm":
        R, C = case["rows"], case["C"]
        wide = C + 40 if case["sliced"] else C
        # activations with a mean of their own and a spread that differs from channel to channel
        x = (torch.randn((R, wide), generator=gen, device=dev) * (0.5 + 2.0 * torch.rand((wide,), generator=gen, device=dev)) + 0.3).to(dtype)
        s["x"] = leaf(x[:, 16:16 + C] if case["sliced"] else x)
        s["gamma"] = leaf(_normal(gen, (C,), torch.float32, 0.1, 1.0)) if case["affine"] else None
        s["beta"] = leaf(_normal(gen, (C,), torch.float32, 0.1)) if case["affine"] else None
        s["dy"] = _normal(gen, (R, C), dtype) if train else None
    elif op == "dropout":
        n = case["n"]
        s["x"] = leaf(_normal(gen, (n,), dtype))
        s["res"] = leaf(_normal(gen, (n,), dtype)) if case["residual"] else None
        s["dy"] = _normal(gen, (n,), dtype) if train else None
        s["seed"] = (int(seed) * 6364136223846793005 + 1442695040888963407) % (1 << 63)
    elif op == "rotary":
        B, H, Hk, D = case["B"], case["H"], case["Hk"], case["D"]
        T = case["t"] * case["h"] * case["w"]
        qkv = _normal(gen, (B, T, (H + 2 * Hk) * D), dtype)   # the fused product that the queries and keys are columns of
        s["q"] = leaf(qkv[..., :H * D].unflatten(-1, (H, D)))
        s["k"] = leaf(qkv[..., H * D:(H + Hk) * D].unflatten(-1, (Hk, D)))
        sizes, sections = (case["t"], case["h"], case["w"]), (case["d_t"], case["d_h"], case["d_w"])
        axes = [a for a in range(3) if sections[a]]
        grid = torch.stack(torch.meshgrid(*[torch.arange(n, device=dev) for n in sizes], indexing="ij"), -1).view(T, 3)[:, axes]
        if case["per_row"]:     # each sample is a crop at an offset of its own
            grid = grid + torch.randint(0, 2048, (B, 1, len(axes)), generator=gen, device=dev)
        s["pos"] = grid.float() * 0.7 if case["scaled"] else grid.to(torch.int32)
        s["sections"] = tuple(sections[a] for a in axes)
        # freqs[j] of a section of n entries: 10000 ** (-2 j / n); the pairs' places in a head and their axes
        freqs, first, second, axis, at = [], [], [], [], 0
        for a, n in enumerate(s["sections"]):
            for j in range(n // 2):
                freqs.append(10000.0 ** (-2.0 * j / n))
                first.append(at + 2 * j if case["interleaved"] else at + j)
                second.append(at + 2 * j + 1 if case["interleaved"] else at + j + n // 2)
                axis.append(a)
            at += n
        s["freqs"] = torch.tensor(freqs, dtype=torch.float64, device=dev)
        s["first"], s["second"], s["axis"] = (torch.tensor(i, device=dev) for i in (first, second, axis))
        s["dq"] = _normal(gen, (B, T, H, D), dtype) if train else None
        s["dk"] = _normal(gen, (B, T, Hk, D), dtype) if train else None
    else:
        B, T, H, Hk, D = (case[n] for n in ("B", "T", "H", "Hk", "D"))
        qkv = _normal(gen, (B, T, (H + 2 * Hk) * D), dtype, 1.3)
        s["q"] = leaf(qkv[..., :H * D].unflatten(-1, (H, D)))
        s["k"] = leaf(qkv[..., H * D:(H + Hk) * D].unflatten(-1, (Hk, D)))
        s["v"] = leaf(qkv[..., (H + Hk) * D:].unflatten(-1, (Hk, D)))
        s["do"] = _normal(gen, (B, T, H, D), dtype) if train else None
        s["lengths"] = None
        if case["ragged"]:
            n = torch.randint((T + 1) // 2, T + 1, (B,), generator=gen, device=dev, dtype=torch.int32)
            n[0] = T
            if B > 3:
                n[1] = 0        # a slot of the batch that no sequence fills
            s["lengths"] = n
    return s


# ---------------------------------------------------------------------------------------------- one pass
def run(s):
    op, train = s["case"]["op"], s["case"]["train"]
    if own:
        if train:
            return _own(op, s)
        with torch.no_grad():
            return _own(op, s)
    with torch.no_grad():
        return {"layer_norm": _plain_layer_norm, "dropout": _plain_dropout, "rotary": _plain_rotary, "attention": _plain_attention}[op](s)


def _own(op, s):
    from indm_amd import ops
    case = s["case"]
    if op == "layer_norm":
        y = ops.layer_norm(s["x"], s["gamma"], s["beta"], EPS)
        if not case["train"]:
            return [y]
        leaves = [s["x"], s["gamma"], s["beta"]] if case["affine"] else [s["x"]]
        return [y, *torch.autograd.grad(y, leaves, s["dy"])]
    if op == "dropout":
        y = ops.dropout(s["x"], case["p"], s["seed"], res=s["res"])
        if not case["train"]:
            return [y]
        return [y, *torch.autograd.grad(y, [s["x"], s["res"]] if case["residual"] else [s["x"]], s["dy"])]
    if op == "rotary":
        q, k = ops.rotary(s["q"], s["k"], s["pos"], s["freqs"], s["sections"], interleaved=case["interleaved"])
        if not case["train"]:
            return [q, k]
        return [q, k, *torch.autograd.grad([q, k], [s["q"], s["k"]], [s["dq"], s["dk"]])]
    o = ops.window_attention(s["q"], s["k"], s["v"], (case["left"], case["right"]), sinks=case["sinks"], causal=case["causal"],
                             lengths=s["lengths"])
    if not case["train"]:
        return [o]
    return [o, *torch.autograd.grad(o, [s["q"], s["k"], s["v"]], s["do"])]


def _plain_layer_norm(s):
    x = s["x"].float()
    d = x - x.mean(-1, keepdim=True)
    rstd = torch.rsqrt((d * d).mean(-1, keepdim=True) + EPS)
    xh = d * rstd
    y = xh * s["gamma"] + s["beta"] if s["gamma"] is not None else xh
    y = y.to(s["x"].dtype)
    if s["dy"] is None:
        return [y]
    dy = s["dy"].float()
    g = dy * s["gamma"] if s["gamma"] is not None else dy
    dx = rstd * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    dx = dx.to(s["x"].dtype)
    return [y, dx] if s["gamma"] is None else [y, dx, (dy * xh).sum(0), dy.sum(0)]


def _philox_words(seed, n, dev):
    """the n first 32-bit words of Philox4x32-10 with the 64-bit key `seed` and the counters 0, 1, 2, ... (int64 values)"""
    low = (1 << 32) - 1
    c0 = torch.arange((n + 3) // 4, device=dev)
    c1 = torch.zeros_like(c0)       # (the counters of these sizes fit 32 bits)
    c2, c3 = torch.zeros_like(c0), torch.zeros_like(c0)
    k0, k1 = seed & low, seed >> 32
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57    # 64-bit products; int64 wraps to the same bits
        c0, c1, c2, c3 = ((p1 >> 32) & low) ^ c1 ^ k0, p1 & low, ((p0 >> 32) & low) ^ c3 ^ k1, p0 & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack([c0, c1, c2, c3], -1).view(-1)[:n]


def _plain_dropout(s):
    p = torch.tensor(s["case"]["p"], dtype=torch.float32)     # the probability as the 32-bit number it is passed as
    keep = (_philox_words(s["seed"], s["x"].numel(), s["x"].device) >> 8) + 1 > float(p) * 2.0 ** 24
    factor = float(1.0 / (1.0 - p))
    y = torch.where(keep, s["x"].float() * factor, 0.0)
    if s["res"] is not None:
        y = y + s["res"].float()
    y = y.to(s["x"].dtype)
    if s["dy"] is None:
        return [y]
    dx = torch.where(keep, s["dy"].float() * factor, 0.0).to(s["x"].dtype)
    return [y, dx] if s["res"] is None else [y, dx, s["dy"]]


def _rotate(x, cos, sin, s, dtype):
    out = x.clone()
    a, b = x[..., s["first"]], x[..., s["second"]]
    out[..., s["first"]] = a * cos - b * sin
    out[..., s["second"]] = b * cos + a * sin
    return out.to(dtype)


def _plain_rotary(s):
    angle = s["pos"].double()[..., s["axis"]] * s["freqs"]    # [T, pairs] or [B, T, pairs]; far positions need 64 bits
    cos, sin = angle.cos().float()[..., None, :], angle.sin().float()[..., None, :]
    dtype = s["q"].dtype
    out = [_rotate(s["q"].float(), cos, sin, s, dtype), _rotate(s["k"].float(), cos, sin, s, dtype)]
    if s["dq"] is None:
        return out
    return out + [_rotate(s["dq"].float(), cos, -sin, s, dtype), _rotate(s["dk"].float(), cos, -sin, s, dtype)]


def _visible(case, lengths, B, dev):
    """[B or 1, 1, T, T]: key j is visible to query i"""
    i = torch.arange(case["T"], device=dev)
    i, j = i[:, None], i[None, :]
    m = ((j >= i - case["left"]) & (j <= i + case["right"])) | (j < case["sinks"])
    if case["causal"]:
        m = m & (j <= i)
    m = m[None]
    if lengths is not None:
        n = lengths.view(B, 1, 1)
        m = m & (i < n) & (j < n)
    return m[:, None]


def _heads_first(x, group=1):
    """[B, T, H, D] -> [B, H * group, T, D], in order"""
    return x.transpose(1, 2).repeat_interleave(group, 1).contiguous()


def _plain_attention(s):
    case, dtype = s["case"], s["q"].dtype
    B, T, H, Hk, D = (case[n] for n in ("B", "T", "H", "Hk", "D"))
    scale, group = 1.0 / math.sqrt(D), H // Hk
    q, k, v = _heads_first(s["q"].float()), _heads_first(s["k"].float(), group), _heads_first(s["v"].float(), group)
    hidden = ~_visible(case, s["lengths"], B, q.device)
    z = (q @ k.transpose(-1, -2).contiguous()).mul_(scale).masked_fill_(hidden, -math.inf)
    top = z.amax(-1, keepdim=True)
    z = z.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = z.sum(-1, keepdim=True)
    p = z.div_(torch.where(total == 0.0, 1.0, total))         # a row that sees nothing gives zeros
    o = (p @ v).transpose(1, 2).to(dtype).contiguous()
    if s["do"] is None:
        return [o]
    do = _heads_first(s["do"].float())
    dv = p.transpose(-1, -2).contiguous() @ do
    dz = do @ v.transpose(-1, -2).contiguous()
    dz = dz.sub_((p * dz).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq = dz @ k
    dk = dz.transpose(-1, -2).contiguous() @ q
    shared = lambda g: g.view(B, Hk, group, T, D).sum(2).transpose(1, 2).to(dtype).contiguous()  # noqa: E731
    return [o, dq.transpose(1, 2).to(dtype).contiguous(), shared(dk), shared(dv)]


# ---------------------------------------------------------------------------------------------- what a pass cannot do without
def _pairs(case):
    """visible query-key pairs of one full sequence"""
    T, sinks = case["T"], min(case["sinks"], case["T"])
    i = torch.arange(T, dtype=torch.int64)
    low, high = torch.clamp(i - case["left"], min=0), torch.clamp(i + case["right"], max=T - 1)
    high = torch.minimum(high, i) if case["causal"] else high
    before = torch.clamp(low, max=sinks)                                              # sinks in front of the window
    after = torch.zeros_like(i) if case["causal"] else torch.clamp(sinks - 1 - high, min=0)   # and behind it
    return int((high - low + 1 + before + after).sum())


def work(case):
    e, twice, op = BYTES[case["dtype"]], 2 if case["train"] else 1, case["op"]
    if op == "layer_norm":
        n = case["rows"] * case["C"]
        return dict(bytes=2 * e * n * twice + (8 * case["C"] * twice if case["affine"] else 0), flops=(8 + (11 if case["train"] else 0)) * n)
    if op == "dropout":
        return dict(bytes=case["n"] * e * (2 * twice + (1 if case["residual"] else 0)), flops=2 * case["n"] * twice)
    T = case["t"] * case["h"] * case["w"] if op == "rotary" else case["T"]
    if op == "rotary":
        n = case["B"] * T * (case["H"] + case["Hk"]) * case["D"]
        axes = sum(case[d] > 0 for d in ("d_t", "d_h", "d_w"))
        return dict(bytes=2 * e * n * twice + 4 * T * axes * (case["B"] if case["per_row"] else 1), flops=3 * n * twice)
    q, kv = case["B"] * T * case["H"] * case["D"], case["B"] * T * case["Hk"] * case["D"]
    # (ragged lengths are data: they are about three quarters of T, and one slot of four or more is empty)
    share = (0.75 if case["B"] <= 3 else 0.75 * (case["B"] - 1) / case["B"]) if case["ragged"] else 1.0
    moved = 2 * q + 2 * kv + (2 * q + 2 * kv if case["train"] else 0)
    return dict(bytes=e * moved * share, flops=(14 if case["train"] else 4) * case["D"] * case["B"] * case["H"] * _pairs(case) * share)


# ---------------------------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "layer_norm":
            return _exact_layer_norm(s)
        if case["op"] == "dropout":
            return _exact_dropout(s)
        if case["op"] == "rotary":
            return _exact_rotary(s)
        return _exact_attention(s)


def _exact_layer_norm(s):
    x, C = s["x"].double(), s["case"]["C"]
    var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
    sd = torch.sqrt(var + EPS)
    unit = (x - mean) / sd
    w = s["gamma"].double() if s["gamma"] is not None else torch.ones(C, dtype=torch.float64, device=x.device)
    y = unit * w + (s["beta"].double() if s["beta"] is not None else 0.0)
    if s["dy"] is None:
        return [y]
    dy = s["dy"].double()
    g = dy * w
    along = (g * unit).sum(1, keepdim=True) / C
    dx = (g - g.sum(1, keepdim=True) / C - unit * along) / sd
    return [y, dx] if s["gamma"] is None else [y, dx, (dy * unit).sum(0), dy.sum(0)]


def _exact_dropout(s):
    import numpy as np
    n, seed = s["case"]["n"], s["seed"]
    # Philox4x32-10 on the host, in unsigned 64-bit words
    ctr = [np.arange((n + 3) // 4, dtype=np.uint64)] + [np.zeros((n + 3) // 4, dtype=np.uint64) for _ in range(3)]
    key, mask = [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF], np.uint64(0xFFFFFFFF)
    for _ in range(10):
        a, b = ctr[0] * np.uint64(0xD2511F53), ctr[2] * np.uint64(0xCD9E8D57)
        ctr = [(b >> np.uint64(32)) ^ ctr[1] ^ np.uint64(key[0]), b & mask, (a >> np.uint64(32)) ^ ctr[3] ^ np.uint64(key[1]), a & mask]
        key = [(key[0] + 0x9E3779B9) % (1 << 32), (key[1] + 0xBB67AE85) % (1 << 32)]
    words = np.stack(ctr, -1).reshape(-1)[:n]
    p = float(np.float32(s["case"]["p"]))
    keep = torch.from_numpy(((words >> np.uint64(8)).astype(np.float64) + 1.0) / 2.0 ** 24 > p).to(s["x"].device)
    y = keep * s["x"].double() / (1.0 - p)
    y = y if s["res"] is None else y + s["res"].double()
    if s["dy"] is None:
        return [y]
    dx = keep * s["dy"].double() / (1.0 - p)
    return [y, dx] if s["res"] is None else [y, dx, s["dy"].double()]


def _exact_rotary(s):
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=s["q"].device), s["pos"].double()[..., s["axis"]] * s["freqs"])
    turn = turn.unsqueeze(-2)

    def turned(x, by):
        x = x.double()
        z = torch.complex(x[..., s["first"]].contiguous(), x[..., s["second"]].contiguous()) * by
        out = x.clone()
        out[..., s["first"]], out[..., s["second"]] = z.real, z.imag
        return out

    out = [turned(s["q"], turn), turned(s["k"], turn)]
    return out if s["dq"] is None else out + [turned(s["dq"], turn.conj()), turned(s["dk"], turn.conj())]


def _exact_attention(s):
    case = s["case"]
    B, T, H, Hk, D = (case[n] for n in ("B", "T", "H", "Hk", "D"))
    group = H // Hk
    q, k, v = (s[n].double() for n in ("q", "k", "v"))
    o = torch.zeros_like(q)
    grads = [torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)] if s["do"] is not None else []
    at = torch.arange(T, device=q.device)
    far = at[None, :] - at[:, None]
    see = ((far >= -case["left"]) & (far <= case["right"])) | (at < case["sinks"])[None, :]
    if case["causal"]:
        see = see & (far <= 0)
    for b in range(B):
        n = T if s["lengths"] is None else int(s["lengths"][b])
        if n == 0:
            continue
        for h in range(H):
            qq, kk, vv = (t.contiguous() for t in (q[b, :n, h], k[b, :n, h // group], v[b, :n, h // group]))
            logits = torch.where(see[:n, :n], qq @ kk.t().contiguous() * D ** -0.5, -math.inf)
            p = torch.softmax(logits, -1)
            o[b, :n, h] = p @ vv
            if grads:
                do = s["do"][b, :n, h].double()
                dp = do @ vv.t().contiguous()
                dl = p * (dp - (o[b, :n, h] * do).sum(-1, keepdim=True)) * D ** -0.5
                grads[0][b, :n, h] = dl @ kk
                grads[1][b, :n, h // group] += dl.t().contiguous() @ qq
                grads[2][b, :n, h // group] += p.t().contiguous() @ do
    return [o] + grads

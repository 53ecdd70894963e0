"""The operators over a quantized cache written out in 64 bits on the CPU (plain loops over sequences and tokens), and
how far float32 kernels may be from them.  Test infrastructure."""
import math

import torch

TOP = {"int8": 127.0, "e4m3": 448.0}
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}   # half a step, relative to the value


def cpu(x):
    return None if x is None else x.detach().cpu()


def clamp(x, lo, hi):
    return max(lo, min(hi, int(x)))


def radians(dims, base=10000.0, scaling=None, factor=1.0, original=None, slow=1.0, fast=32.0):
    """of every pair a position, and the magnitude"""
    out = []
    for p in range(dims // 2):
        b = base * factor ** (dims / (dims - 2)) if scaling == "base" else base
        w = b ** (-2.0 * p / dims)
        if scaling == "linear":
            w /= factor
        if scaling == "bands":
            keep = clamp01((original * w / (2 * math.pi) - slow) / (fast - slow))
            w = w * (keep + (1 - keep) / factor)
        out.append(w)
    return torch.tensor(out, dtype=torch.float64), 0.1 * math.log(factor) + 1 if scaling == "bands" else 1.0


def clamp01(x):
    return max(0.0, min(1.0, x))


def angles(turns, positions):
    """turns int64 [pairs] (2^-64 of a turn), positions int64 [..] -> radians [.., pairs], the whole turns dropped exactly"""
    f = positions[..., None] * turns   # mod 2^64, as whole numbers
    return f.double() * (2.0 ** -63 * math.pi)


def rotated(x, positions, rotary):
    """x [heads, n, dk] in 64 bits, positions [n]"""
    turns, magnitude, interleaved = rotary
    a = angles(cpu(turns), positions.long())
    c, s = a.cos() * magnitude, a.sin() * magnitude
    y, half = x.double().clone(), turns.numel()
    i = torch.arange(half)
    ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    va, vb = y[..., ia].clone(), y[..., ib].clone()
    y[..., ia], y[..., ib] = va * c - vb * s, va * s + vb * c
    return y


def lineage(parents, n):
    """for each new token the set of those it sees; parents None: a chain"""
    seen = []
    for i in range(n):
        p = i - 1 if parents is None else int(parents[i])
        seen.append((seen[p] if 0 <= p < i else set()) | {i})
    return seen


def quotients(x, format):
    """float32 rows -> exact codes' steps before rounding (64 bits), the size of a step relative to the scale, the largest magnitudes"""
    most = x.abs().amax(-1, keepdim=True).double()
    t = x.double() * TOP[format] / torch.where(most > 0, most, torch.ones_like(most))
    step = torch.ones_like(t) if format == "int8" else torch.exp2((torch.frexp(t)[1] - 1).clamp_min(-6).double() - 3)
    return t / step, step, most[..., 0]


def coded(x, format):
    """values of the codes (float64), scales (float32), and where the quotient is within 1e-6 of a border of two codes without being a
    tie: there a key turned in another order of operations may take the other one"""
    bad = ~torch.isfinite(x).all(-1)
    q, step, most = quotients(torch.where(bad[..., None], torch.zeros_like(x), x), format)
    near = ((q - q.floor() - 0.5).abs() < 1e-6) & (q - q.floor() != 0.5)
    scale = (most.float().numpy() / torch.tensor(TOP[format]).float().numpy())
    scale = torch.from_numpy(scale).clone()
    scale[bad] = math.nan
    return q.round() * step, scale, near


def append(cache, k, v, lens, parents, counts, rotary, format):
    """cache: (code values float64 [S, H, cap, dk] k, v, scales k, v) on the CPU, written in place; returns where a code may differ (k)"""
    kc, vc, ks, vs = cache
    S, H, n, dk = k.shape
    cap, near = kc.shape[2], torch.zeros_like(kc, dtype=torch.bool)
    for s in range(S):
        length, m = clamp(lens[s], 0, cap), n if counts is None else clamp(counts[s], 0, n)
        seen = lineage(None if parents is None else parents[s], n)
        at = torch.tensor([length + len(t) - 1 for t in seen])
        rows = k[s].float() if rotary is None else rotated(k[s], at, rotary).float()
        for dst, scales, x, is_key in ((kc, ks, rows, True), (vc, vs, v[s].float(), False)):
            values, scale, close = coded(x, format)
            for i in range(min(m, cap - length)):
                dst[s, :, length + i] = values[:, i]
                scales[s, :, length + i] = scale[:, i]
                if is_key and rotary is not None:
                    near[s, :, length + i] = close[:, i]
    return near


def attention(q, kc, vc, ks, vs, lens, parents, counts, scale):
    """-> (result, how far a kernel's may be) [S, H, n, dk] float64; cache as code values float64 and float32 scales"""
    S, H, n, dk = q.shape
    heads, cap = kc.shape[1], kc.shape[2]
    group = H // heads
    out, tol = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    one = q.dtype != torch.float32
    for s in range(S):
        length, m = clamp(lens[s], 0, cap), n if counts is None else clamp(counts[s], 0, n)
        seen = lineage(None if parents is None else parents[s], n)
        for i in range(m):
            at = list(range(length)) + [length + j for j in sorted(seen[i]) if length + j < cap]
            if not at:
                continue
            for h in range(heads):
                K = kc[s, h, at] * ks[s, h, at].double()[:, None]
                V = vc[s, h, at] * vs[s, h, at].double()[:, None]
                Q = q[s, h * group:(h + 1) * group, i].double()
                e = scale * (Q @ K.t())
                p = torch.softmax(e, -1)
                out[s, h * group:(h + 1) * group, i] = p @ V
                tol[s, h * group:(h + 1) * group, i] = bound(Q, K, V, vs[s, h, at].double(), p, e, scale, one)
    return out, tol + out.abs() * HALF[q.dtype]


def bound(Q, K, V, v_scale, p, e, scale, one):
    """Of a result, before it is rounded to its type.  d: how far the logarithm of a weight may be off - the products' sum
    (dk + 4 roundings of 2^-23, the matrix units' included, a query in 22 bits, factors), the logarithm's own size (the subtraction and
    the exponential's argument, 4 roundings of it), the exponential (2^-22).  A weight is off by d, and by its rounding to 11 or 22
    bits, or where it is small by half a step of the smallest float16 at a unit of 2^9, over a carried scale of up to
    the largest; its sum likewise without the rounding; sums over the positions add half a step each."""
    n, dk = K.shape
    products = scale * (Q.abs() @ K.abs().t())
    d = products.amax(-1) * (dk + 8) * 2.0 ** -23 + e.abs().amax(-1) * 2.0 ** -21 + 2.0 ** -21 + n * 2.0 ** -24
    size = p @ V.abs()                        # [rows, dk]
    rounding = 2.0 ** -11 if one else 2.0 ** -22
    # a float16 down to 2^-24 in steps of 2^-24, with a second one of the remainder down to it, too
    smallest = 2.0 ** -25 / 2.0 ** 9 * v_scale.max() * (V.abs() / torch.where(v_scale > 0, v_scale, torch.ones_like(v_scale))[:, None]).sum(0)
    top = p.amax(-1, keepdim=True)            # (weights are relative to the largest)
    return size * (2 * d[:, None] + rounding + n * 2.0 ** -24) + top * smallest * 16

"""The operators over a cache in pages, and the verification of drafted tokens, written out in 64 bits on the CPU (plain loops over
sequences and tokens), and how far the kernels may be from them.  Test infrastructure."""
import torch

from cache_oracle import HALF, clamp, cpu


def ceil(a, b):
    return -(-a // b)


def reserve(table, held, free, count, lens, n, page, counts=None):
    """table [S][row], held [S], free [pages], count [1] as lists, changed in place -> slots [S][n]"""
    S, row, pages = len(table), len(table[0]) if table else 0, len(free)
    available, dealt, out = clamp(count[0], 0, pages), 0, []
    taken = 0
    for s in range(S):
        m = n if counts is None else clamp(counts[s], 0, n)
        have = clamp(held[s], 0, row)
        need = ceil(max(lens[s], 0) + m, page)
        more = 0 if need > row else max(0, need - have)
        dealt += more
        if more and dealt <= available:
            for j in range(more):
                table[s][have + j] = free[available - 1 - (dealt - more + j)]
            held[s], taken = have + more, dealt
    count[0] = available - taken
    for s in range(S):
        m = n if counts is None else clamp(counts[s], 0, n)
        line = []
        for i in range(n):
            at = max(lens[s], 0) + i
            p = table[s][at // page] if at // page < row else -1
            line.append(p * page + at % page if i < m and 0 <= p < pages else -1)
        out.append(line)
    return out


def trim(table, held, free, count, lens, page):
    S, row, pages = len(table), len(table[0]) if table else 0, len(free)
    available, gone = clamp(count[0], 0, pages), []
    for s in range(S):
        have = clamp(held[s], 0, row)
        keep = min(have, ceil(max(lens[s], 0), page))
        gone += table[s][keep:have]
        table[s][keep:have] = [-1] * (have - keep)
        held[s] = keep
    for t, p in enumerate(gone):
        to = available + len(gone) - 1 - t
        if to < pages:
            free[to] = p
    count[0] = min(available + len(gone), pages)


def attention(q, k, v, table, lens, counts, scale):
    """q [S, H, n, dk], k, v [pages, heads, page, dk], table [S, row] on the CPU -> (result, how far a kernel's may be) in 64 bits"""
    S, H, n, dk = q.shape
    pages, heads, page = k.shape[:3]
    group, row = H // heads, table.shape[1]
    out, tol = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for s in range(S):
        m = n if counts is None else clamp(counts[s], 0, n)
        past = clamp(lens[s], 0, row * page)
        at = torch.arange(min(past + m, row * page))
        ids = table[s].long()[at // page]
        there = (ids >= 0) & (ids < pages)
        at, ids = at[there], ids[there]
        for h in range(heads):
            K, V = k[ids, h, at % page].double(), v[ids, h, at % page].double()
            for i in range(m):
                seen = int((at <= past + i).sum())
                if seen == 0:
                    continue
                Q = q[s, h * group:(h + 1) * group, i].double()
                e = scale * (Q @ K[:seen].t())
                p = torch.softmax(e, -1)
                out[s, h * group:(h + 1) * group, i] = p @ V[:seen]
                tol[s, h * group:(h + 1) * group, i] = bound(Q, K[:seen], V[:seen], p, e, scale, q.dtype)
    return out, tol + out.abs() * HALF[q.dtype]


def bound(Q, K, V, p, e, scale, dtype):
    """Of a result, before it is rounded to its type.  d: how far the logarithm of a weight may be off - the products' sum (dk + 8
    roundings of 2^-23, the matrix units' included), the logarithm's own size (factor, subtraction and the exponential's argument, 4 roundings
    of it), the exponential (2^-22).  A weight is off by d, its sum likewise; it is rounded to the type ahead of the product with the
    values (float16: down to half a step of 2^-24 at a unit of 2^11); sums over the positions add a rounding of 2^-23 each."""
    n, dk = K.shape
    products = scale * (Q.abs() @ K.abs().t())
    d = products.amax(-1) * (dk + 8) * 2.0 ** -23 + e.abs().amax(-1) * 2.0 ** -21 + 2.0 ** -21
    size = p @ V.abs()
    rounding = 0.0 if dtype == torch.float32 else HALF[dtype]
    small = 2.0 ** -36 * V.abs().sum(0) if dtype == torch.float16 else 0.0
    return size * (2 * d[:, None] + rounding + (n + 8) * 2.0 ** -23) + p.amax(-1, keepdim=True) * small


def verify(tokens, target, random, draft=None, parents=None, counts=None):
    """tokens [S][n], target [S, n, vocab] .. on the CPU -> path [S][n], accepted [S], next [S], and how near a number came to a border
    (relative to what it is held against)"""
    S, n, vocab = target.shape
    paths, accepted, following, near = [], [], [], 1.0

    def mass(x):
        return torch.where(x > 0, x, torch.zeros_like(x))
    for s in range(S):
        m = n if counts is None else clamp(counts[s], 0, n)
        if m == 0:
            paths.append([-1] * n)
            accepted.append(0)
            following.append(-1)
            continue
        path, here, refused, gone = [0], 0, [], 0.0
        for i in range(1, m):
            parent = i - 1 if parents is None else int(parents[s][i])
            if parent != here or parent >= i:
                continue
            t, u = int(tokens[s][i]), float(random[s][i])
            p = float(mass(target[s, here, t].double())) if 0 <= t < vocab and t not in refused else 0.0
            q = 1.0 - gone if draft is None else float(mass(draft[s, here, t].double())) if 0 <= t < vocab else 1.0
            if p > 0:
                near = min(near, abs(u * q - p) / p)
            if u * q < p:
                path.append(i)
                here, refused, gone = i, [], 0.0
            else:
                refused.append(t)
                gone += p
        own = mass(target[s, here].double())
        left = own.clone()
        if refused and draft is not None:
            left = mass(own - mass(draft[s, here].double()))
        elif refused:
            for t in refused:
                if 0 <= t < vocab:
                    left[t] = 0
        if left.sum() <= 0:
            left = own
        sums = left.cumsum(0)
        bar = float(random[s][0]) * float(sums[-1])
        above = (sums > bar).nonzero()
        near = min(near, float((sums - bar).abs().min() / sums[-1])) if sums[-1] > 0 else near
        following.append(int(above[0]) if len(above) else -1)
        paths.append(path + [-1] * (n - len(path)))
        accepted.append(len(path))
    return paths, accepted, following, near


__all__ = ["attention", "bound", "cpu", "reserve", "trim", "verify"]

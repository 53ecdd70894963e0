"""Rotary positions, the cache in 8 bits and the attention over it on the GPU, against the same written out in 64 bits on
the CPU (cache_oracle.py, which says how far results may be)."""
import math
import threading

import pytest
import torch

import cache_oracle as oracle
from conftest import load

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def say(*a):
    print(*a, flush=True)


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def maker(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return lambda *s: torch.randn(*s, device="cuda", generator=g)


def side_by_side(r, S, H, n, dk, dtype):
    return r(S, n, H, dk).to(dtype).transpose(1, 2)


def same(a, b):
    return a.shape == b.shape and a.dtype == b.dtype and torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def check(got, want, tol):
    got = got.cpu().double()
    bad = ~((got - want).abs() <= tol) & ~(torch.isnan(got) & torch.isnan(want))
    assert not bad.any(), "%d of %d off, first at %s: %r, %r +- %r" % (
        bad.sum(), bad.numel(), bad.nonzero()[0].tolist(), got[bad][0].item(), want[bad][0].item(), tol[bad][0].item())


def filled(r, S, H, cap, dk, format, spread=1.0):
    """a cache of random codes and scales"""
    kv = load("cache")
    cache = kv.newCache(S, H, cap, dk, format)
    for codes, scales in ((cache.k, cache.kScale), (cache.v, cache.vScale)):
        x = r(S, H, cap, dk)
        top = x.abs().amax(-1)
        y = x / top[..., None] * oracle.TOP[format]
        codes.copy_(y.round().to(torch.int8) if format == "int8" else y.to(torch.float8_e4m3fn))
        scales.copy_(top / oracle.TOP[format] * torch.exp(spread * r(S, H, cap)))
    return cache


def on_cpu(cache):
    """code values in 64 bits, and scales"""
    return [cache.k.float().cpu().double(), cache.v.float().cpu().double(), cache.kScale.cpu(), cache.vScale.cpu()]


def expected(q, cache, lens, parents=None, counts=None, scale=None):
    kc, vc, ks, vs = on_cpu(cache)
    return oracle.attention(q.cpu(), kc, vc, ks, vs, lens.cpu(), oracle.cpu(parents), oracle.cpu(counts), scale or q.shape[-1] ** -0.5)


# ---- rotary positions ------------------------------------------------------------------------------------
def rotary_tolerance(x, rotary, want, dtype):
    """sine and cosine in float32 with the angle's own rounding (2^-22 together), two products and a sum (2^-23)"""
    size = x.double().abs()
    return 3 * 2.0 ** -22 * rotary.magnitude * size.amax(-1, keepdim=True) * 2 + want.abs() * oracle.HALF[dtype]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("S,H,n,dk,dims,interleaved,scaling", [
    (1, 1, 1, 16, 16, False, None), (4, 16, 1, 64, 64, False, None), (2, 5, 7, 80, 40, True, "bands"), (3, 8, 33, 128, 64, False, "linear"),
    (2, 3, 129, 256, 256, True, "base"), (1, 6, 4, 96, 8, False, "bands"), (2, 33, 520, 64, 32, False, None)])
def test_rotary(dtype, S, H, n, dk, dims, interleaved, scaling):
    kv, r = load("cache"), maker(S + n)
    rotary = kv.makeRotary(dims, interleaved=interleaved, scaling=scaling, factor=4.0 if scaling else 1.0, original=512)
    x = side_by_side(r, S, H, n, dk, dtype)
    first = [(-7, 0, 100000, 2 ** 31 - 1 - n)[s % 4] for s in range(S)]
    at = torch.tensor(first)[:, None] + torch.arange(n)
    want = torch.stack([oracle.rotated(x[s].cpu(), at[s], rotary) for s in range(S)])
    tol = rotary_tolerance(x.cpu(), rotary, want, dtype)
    got = kv.rotaryPositions(x, ints(first), rotary)
    assert got.shape == x.shape and got.transpose(1, 2).is_contiguous() and got.dtype == dtype
    check(got, want, tol)
    assert same(got[..., dims:], x[..., dims:])
    # positions of every row; head by head; in place; into another tensor; tensors that have to be copied first
    assert same(kv.rotaryPositions(x, at.to(torch.int32).cuda(), rotary), got)
    assert same(kv.rotaryPositions(x.contiguous(), at.cuda(), rotary), got)
    out = torch.zeros(S, H, n, 2 * dk, dtype=dtype, device="cuda")[..., dk:]
    assert kv.rotaryPositions(x, ints(first), rotary, out).data_ptr() == out.data_ptr() and same(out, got)
    y = x.clone()
    assert kv.rotaryPositions(y, ints(first), rotary, y).data_ptr() == y.data_ptr() and same(y, got)
    odd = torch.zeros(S * H * n * dk + 1, dtype=dtype, device="cuda")[1:].view(S, H, n, dk).copy_(x)
    assert same(kv.rotaryPositions(odd, ints(first), rotary), got)
    wide = torch.zeros(S, H, n, dk + 1, dtype=dtype, device="cuda")[..., :dk].copy_(x)
    assert same(kv.rotaryPositions(wide, ints(first), rotary), got)
    assert same(kv.rotaryPositions(x[:, :1].expand(S, H, n, dk), ints(first), rotary)[:, H - 1], got[:, 0])


def test_rotary_of_nothing_and_refusals():
    kv, error, r = load("cache"), load("_lib").MarianHipError, maker(1)
    rotary = kv.makeRotary(32)
    x = side_by_side(r, 2, 4, 3, 64, F32)
    assert kv.rotaryPositions(x[:, :, :0], ints([1, 2]), rotary).shape == (2, 4, 0, 64)
    assert kv.rotaryPositions(x[:0], ints([]), rotary).shape == (0, 4, 3, 64)
    for bad in (lambda: kv.rotaryPositions(x.double(), ints([1, 2]), rotary), lambda: kv.rotaryPositions(x, ints([1]), rotary),
                lambda: kv.rotaryPositions(x, ints([1, 2]).float(), rotary), lambda: kv.rotaryPositions(x[..., :24], ints([1, 2]), rotary),
                lambda: kv.rotaryPositions(x, ints([1, 2]), kv.makeRotary(128)), lambda: kv.rotaryPositions(x, ints([1, 2]).cpu(), rotary),
                lambda: kv.rotaryPositions(x, ints([1, 2]), kv.makeRotary(32, device="cpu")), lambda: kv.rotaryPositions(x[0], ints([1, 2]), rotary),
                lambda: kv.rotaryPositions(x, ints([1, 2]), rotary, x.contiguous()[:, :, :2]),
                lambda: kv.rotaryPositions(x[:, :, :2], ints([1, 2]), rotary, x[:, :, 1:])):
        with pytest.raises(error):
            bad()


# ---- writing and reading ------------------------------------------------------------------------------------
def check_written(cache, want, near, before, lens, counts, n):
    """codes and scales are the expected ones (next to a border a code may be the next one), and all other rows are as before"""
    S, H, cap, dk = cache.k.shape
    kc, vc, ks, vs = on_cpu(cache)
    written = torch.zeros(S, 1, cap, dtype=torch.bool)
    for s in range(S):
        first = oracle.clamp(lens[s], 0, cap)
        written[s, 0, first:first + (n if counts is None else oracle.clamp(counts[s], 0, n))] = True
    rows = written.expand(S, H, cap)
    for got, right, close in ((kc, want[0], near), (vc, want[1], torch.zeros_like(near))):
        off = (got != right) & rows[..., None]
        assert not (off & ~close).any(), "%d codes differ" % (off & ~close).sum()
        assert not off.any() or (got - right)[off].abs().max() <= 32
    for got, right in ((ks, want[2]), (vs, want[3])):
        g, w = got[rows], right[rows]
        # (a row's largest value, turned in 64 bits in another order, may round to the next float32; the quotient's half step)
        assert torch.equal(torch.isnan(g), torch.isnan(w)) and bool(((g - w).abs() <= w.abs() * 2.0 ** -22)[~torch.isnan(w)].all())
    for t, b in zip(cache, before):
        a = t.view(torch.uint8).view(S, H, cap, -1).cpu()[~rows]
        assert torch.equal(a, b.view(torch.uint8).view(S, H, cap, -1).cpu()[~rows])


@pytest.mark.parametrize("dtype,format", [(F32, "int8"), (F32, "e4m3"), (F16, "int8"), (BF16, "e4m3")])
@pytest.mark.parametrize("S,H,G,n,cap,dk,dims,interleaved,tree", [
    (1, 1, 1, 1, 1, 16, 0, False, False), (5, 16, 1, 1, 9, 64, 64, False, False), (3, 2, 4, 13, 40, 80, 40, True, True),
    (2, 3, 2, 64, 70, 128, 128, False, True), (4, 1, 8, 37, 50, 256, 64, True, False), (2, 2, 1, 6, 20, 96, 96, False, False)])
def test_append(dtype, format, S, H, G, n, cap, dk, dims, interleaved, tree):
    kv, r = load("cache"), maker(7 * S + n)
    rotary = kv.makeRotary(dims, interleaved=interleaved, scaling="bands", factor=2.0, original=64) if dims else None
    k, v, q = (side_by_side(r, S, h, n, dk, dtype) for h in (H, H, G * H))
    lens = ints([(cap - n, 0, cap - 1, -3, cap + 5)[s % 5] for s in range(S)])
    counts = ints([(n, n + 3, n // 2, -1, 1)[s % 5] for s in range(S)])
    parents = torch.randint(-2, n + 2, (S, n), device="cuda", dtype=torch.int32) if tree else None
    if tree:   # a tree that goes deep, too
        parents[0] = torch.arange(n, device="cuda") - 1
    for given in (counts, None):
        cache = filled(r, S, H, cap, dk, format)
        before, want = [t.clone() for t in cache], on_cpu(cache)
        near = oracle.append(want, k.cpu(), v.cpu(), lens.cpu(), oracle.cpu(parents), oracle.cpu(given), rotary, format)
        kept = [t.clone() for t in (k, v, q)]
        got = kv.appendToCache(cache, k, v, lens, parents, given, rotary, q)
        check_written(cache, want, near, before, lens.tolist(), None if given is None else given.tolist(), n)
        assert all(same(a, b) for a, b in zip(kept, (k, v, q)))
        # queries
        assert got.shape == q.shape and got.transpose(1, 2).is_contiguous()
        for s in range(S):
            m = n if given is None else oracle.clamp(given[s], 0, n)
            at = torch.tensor([oracle.clamp(lens[s], 0, cap) + len(t) - 1 for t in oracle.lineage(None if parents is None else parents[s].cpu(), n)])
            turned = q[s].cpu().double() if rotary is None else oracle.rotated(q[s].cpu(), at, rotary)
            # (float16 has steps of 2^-24 at the least)
            check(got[s, :, :m], turned[:, :m], turned[:, :m].abs() * (oracle.HALF[dtype] + 2.0 ** -23) + (2.0 ** -25 if dtype == F16 else 0.0))
            assert not got[s, :, m:].any()
        # without queries, and with queries in place, on the same cache
        again = kv.KeyValueCache(*(t.clone() for t in before))
        assert kv.appendToCache(again, k.contiguous(), v, lens.long(), parents, given, rotary) is None
        assert all(same(a, b) for a, b in zip(again, cache))
        turned = q.clone()
        assert kv.appendToCache(again, k, v, lens, parents, given, rotary, turned, turned).data_ptr() == turned.data_ptr()
        assert same(turned, got) and all(same(a, b) for a, b in zip(again, cache))


def test_ties_go_to_the_even_code():
    kv = load("cache")
    # int8: largest 127 * 2^k, so that halves are exact quotients; e4m3: largest 448 * 2^k, halfway between two steps of every binade
    row = torch.zeros(64)
    row[0] = 127.0
    row[1:64] = torch.arange(-31, 32) + 0.5
    for k in (-40, 0, 30):
        cache = kv.newCache(1, 1, 1, 64, "int8")
        x = (row * 2.0 ** k).view(1, 1, 1, 64).cuda()
        kv.appendToCache(cache, x, -x, ints([0]))
        assert torch.equal(cache.k.view(-1).cpu().float(), row.round()) and torch.equal(cache.v.view(-1).cpu().float(), (-row).round())
        assert cache.kScale.item() == 2.0 ** k
    steps = [m * 2.0 ** e for e in range(-6, 9) for m in (8.5, 9.5, 14.5, 15.5)] + [0.5, 1.5, 6.5, 7.5]
    units = torch.tensor(steps[:60]) * 2.0 ** -3   # in units of 2^-3 a binade: quotients m 2^(e - 3)
    row = torch.zeros(64)
    row[0] = 448.0
    row[1:61] = units[:60]
    row[61:64] = torch.tensor([0.5, 1.5, 6.5]) * 2.0 ** -9
    cache = kv.newCache(1, 1, 1, 64, "e4m3")
    x = row.view(1, 1, 1, 64).cuda()
    kv.appendToCache(cache, x, x, ints([0]))
    q, step, _ = oracle.quotients(row.view(1, 64), "e4m3")
    want = (q.round() * step).clamp(max=448.0)
    assert torch.equal(cache.k.view(1, 64).float().cpu().double(), want)


@pytest.mark.parametrize("format", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_rows_of_zeros_and_rows_that_are_not_finite(format, dtype):
    kv, r = load("cache"), maker(3)
    x = r(1, 2, 8, 64).to(dtype)
    x[0, 0, 0] = 0.0
    x[0, 0, 1, 5] = math.nan
    x[0, 0, 2, 63] = math.inf
    x[0, 0, 3, 0] = -math.inf
    x[0, 0, 4] *= 1e-6 if dtype == F16 else 1e-30
    x[0, 0, 5] *= 1e4 if dtype == F16 else 1e30
    x[0, 0, 6] = -0.0
    cache = kv.newCache(1, 2, 8, 64, format)
    want = on_cpu(cache)
    oracle.append(want, x.cpu(), x.cpu(), [0], None, None, None, format)
    kv.appendToCache(cache, x, x, ints([0]))
    assert torch.equal(cache.k.float().cpu().double(), want[0]) and torch.equal(cache.v.float().cpu().double(), want[1])
    assert torch.isnan(cache.kScale[0, 0]).tolist() == [False, True, True, True, False, False, False, False]
    assert cache.kScale[0, 0, 0] == 0 and cache.kScale[0, 0, 6] == 0
    k, v = kv.readCache(cache, ints([0]), 8, F32)
    assert torch.isnan(k[0, 0]).all(-1).tolist() == [False, True, True, True, False, False, False, False]
    assert not torch.isnan(k[0, 1]).any() and not k[0, 0, 0].any() and same(k, v)


@pytest.mark.parametrize("format", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("S,H,cap,dk,n", [(1, 1, 1, 16, 1), (3, 2, 50, 80, 7), (2, 5, 300, 128, 301), (4, 8, 33, 64, 33), (2, 1, 40, 256, 9), (2, 2, 9, 64, 0)])
def test_read(format, dtype, S, H, cap, dk, n):
    kv, r = load("cache"), maker(n)
    cache = filled(r, S, H, cap, dk, format)
    first = [(0, cap - 3, -2, cap + 4)[s % 4] for s in range(S)]
    kc, vc, ks, vs = on_cpu(cache)
    k, v = kv.readCache(cache, ints(first), n, dtype)
    assert k.dtype == dtype and k.shape == (S, H, n, dk) and v.shape == k.shape
    for got, codes, scales in ((k, kc, ks), (v, vc, vs)):
        for s in range(S):
            for i in range(n):
                p = first[s] + i
                want = (codes[s, :, p] * scales[s, :, p, None].double()) if 0 <= p < cap else torch.zeros(H, dk, dtype=torch.float64)
                # (the product rounded to float32, then to the type; float16 has steps of 2^-24 at the least)
                check(got[s, :, i], want, want.abs() * (oracle.HALF[dtype] + 2.0 ** -24) + (2.0 ** -25 if dtype == F16 else 0.0))


# ---- attention ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,format", [(F32, "int8"), (F32, "e4m3"), (F16, "int8"), (F16, "e4m3"), (BF16, "int8"), (BF16, "e4m3")])
@pytest.mark.parametrize("S,H,G,n,lens,dk,tree", [
    (1, 1, 1, 1, [0], 64, False), (3, 2, 1, 1, [0, 1, 31], 64, False), (2, 3, 4, 1, [32, 33], 128, False), (4, 2, 8, 1, [127, 128, 129, 500], 80, False),
    (2, 1, 16, 1, [64, 700], 256, False), (2, 2, 2, 5, [40, 3], 96, False), (1, 2, 1, 150, [20], 64, False), (2, 1, 3, 70, [0, 129], 128, False),
    (2, 2, 1, 64, [100, 0], 64, True), (3, 1, 4, 17, [0, 31, 200], 128, True), (2, 1, 8, 33, [95, 160], 48, True), (1, 1, 2, 40, [60], 256, True)])
def test_attention(dtype, format, S, H, G, n, lens, dk, tree):
    kv, r = load("cache"), maker(S * n + dk)
    cap = max(lens) + n + 3
    cache = filled(r, S, H, cap, dk, format, 0.5)
    lens = ints(lens)
    q = side_by_side(r, S, H * G, n, dk, dtype)
    parents = torch.randint(-1, n, (S, n), device="cuda", dtype=torch.int32) if tree else None
    if tree:
        i = torch.arange(n, device="cuda", dtype=torch.int32)
        parents = torch.where(parents >= i, i - 1, parents)
    for s in range(S):   # what lies behind the sequence, which nobody may see
        end = int(lens[s]) + n
        for codes, scales in ((cache.k, cache.kScale), (cache.v, cache.vScale)):
            codes.view(torch.uint8)[s, :, end:] = 0x7f
            scales[s, :, end:] = math.nan
    want, tol = expected(q, cache, lens, parents)
    got = kv.AttentionOverCache(q, cache, lens, parents)
    assert got.shape == q.shape and got.transpose(1, 2).is_contiguous() and got.dtype == dtype
    check(got, want, tol)
    assert same(kv.AttentionOverCache(q, cache, lens, parents), got)
    # head by head, and into a tensor that is there
    out = torch.full((S, H * G, n, 2 * dk), 7.0, dtype=dtype, device="cuda")
    assert kv.AttentionOverCache(q.contiguous(), cache, lens.long(), parents, out=out[..., :dk]).data_ptr() == out.data_ptr()
    assert same(out[..., :dk], got) and bool((out[..., dk:] == 7.0).all())
    # only some of the tokens are there
    counts = ints([(n // 2, 0, n + 9, 1)[s % 4] for s in range(S)])
    want, tol = expected(q, cache, lens, parents, counts)
    check(kv.AttentionOverCache(q, cache, lens, parents, counts), want, tol)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("S,H,G,n,dk,lens", [(1, 1, 1, 1, 64, [20000]), (2, 2, 8, 1, 128, [9001, 300]), (3, 1, 4, 6, 128, [5, 6007, 0]), (1, 2, 2, 40, 64, [4097]),
                                             (70, 1, 1, 1, 64, [i * 7 + (3000 if i == 66 else 0) for i in range(70)]), (1, 1, 2, 2, 256, [7000])])
def test_positions_split_over_workgroups(dtype, S, H, G, n, dk, lens):
    kv, r = load("cache"), maker(S + dk)
    cache = filled(r, S, H, max(lens) + n, dk, "int8", 0.3)
    q = side_by_side(r, S, H * G, n, dk, dtype)
    want, tol = expected(q, cache, ints(lens))
    got = kv.AttentionOverCache(q, cache, ints(lens))
    check(got, want, tol)
    for _ in range(3):   # (the counters are back at zero)
        assert same(kv.AttentionOverCache(q, cache, ints(lens)), got)
    short = ints([l // 3 for l in lens])
    check(kv.AttentionOverCache(q, cache, short), *expected(q, cache, short))
    assert same(kv.AttentionOverCache(q, cache, ints(lens)), got)


def test_more_sequences_than_a_wave_has_lanes_and_many_heads():
    kv, r = load("cache"), maker(11)
    S, H, dk = 333, 2, 64
    lens = [(i * 37) % 200 for i in range(S)]
    cache = filled(r, S, H, 210, dk, "e4m3", 0.2)
    q = side_by_side(r, S, 2 * H, 1, dk, F16)
    check(kv.AttentionOverCache(q, cache, ints(lens)), *expected(q, cache, ints(lens)))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("format", ["int8", "e4m3"])
def test_what_a_token_does_not_see_does_not_matter(dtype, format):
    """Drafted tokens of other branches whose rows are NaN, or enormous: not in the results of those that do not see them"""
    kv, r = load("cache"), maker(5)
    n, length, dk = 8, 40, 64
    parents = ints([[-1, 0, 0, 1, -1, 4, 4, 2]])
    cache = filled(r, 1, 1, length + n, dk, format, 0.2)
    q = side_by_side(r, 1, 2, n, dk, dtype)
    lens = ints([length])
    want = kv.AttentionOverCache(q, cache, lens, parents)
    check(want, *expected(q, cache, lens, parents))
    for value in (math.nan, 1e30, 0.0):
        for kind in (cache.kScale, cache.vScale):
            saved = kind[0, 0, length + 4].item()
            kind[0, 0, length + 4] = value
            got = kv.AttentionOverCache(q, cache, lens, parents)
            blind = [0, 1, 2, 3, 7]   # (tokens 4, 5 and 6 see token 4)
            check(got[:, :, blind], *(t[:, :, blind] for t in expected(q, cache, lens, parents)))
            if math.isnan(value):
                assert torch.isnan(got[:, :, [4, 5, 6]]).all() and not torch.isnan(got[:, :, blind]).any()
            kind[0, 0, length + 4] = saved
    assert same(kv.AttentionOverCache(q, cache, lens, parents), want)
    # a settled position that is NaN is in all of them
    cache.vScale[0, 0, 3] = math.nan
    assert torch.isnan(kv.AttentionOverCache(q, cache, lens, parents)).all()


def test_queries_that_are_not_finite_and_queries_of_all_sizes():
    kv, r = load("cache"), maker(6)
    cache = filled(r, 1, 1, 100, 64, "int8", 0.2)
    for dtype in (F32, F16, BF16):
        q = r(1, 8, 1, 64).to(dtype)
        q[0, 1, 0, 3] = math.nan
        q[0, 2, 0, 63] = math.inf
        q[0, 3] = 0.0
        q[0, 4] *= 1e-5 if dtype == F16 else 1e-37
        q[0, 5] *= 1e-3
        q[0, 6] *= 100.0
        got = kv.AttentionOverCache(q, cache, ints([99]))
        assert torch.isnan(got[0, [1, 2]]).all()
        keep = [0, 3, 4, 5, 6, 7]
        check(got[:, keep], *expected(q[:, keep], cache, ints([99])))
        assert same(kv.AttentionOverCache(q[:, keep].contiguous(), cache, ints([99])), got[:, keep].contiguous())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scales_of_all_sizes(dtype):
    """Values whose scales grow and fall by powers of ten along the sequence, keys that make late positions heavy"""
    kv, r = load("cache"), maker(8)
    cap, dk = 600, 128
    cache = filled(r, 2, 2, cap, dk, "int8", 0.0)
    i = torch.arange(cap, device="cuda").float()
    cache.vScale[0] = 10.0 ** (i / 100 - 3)
    cache.vScale[1] = 10.0 ** (3 - i / 100)
    cache.kScale[0] *= i / 300
    cache.vScale[1, 1, :64] = 0.0
    q = side_by_side(r, 2, 8, 3, dk, dtype) * 2
    check(kv.AttentionOverCache(q, cache, ints([cap - 3, 200])), *expected(q, cache, ints([cap - 3, 200])))


def test_tokens_past_the_capacity():
    """What does not fit is dropped by the write and not seen by the attention; a token that sees nothing gives zeros"""
    kv, r = load("cache"), maker(9)
    cache = kv.newCache(2, 1, 4, 64)
    x = r(2, 1, 3, 64)
    lens = ints([2, 0])
    before = [t.clone() for t in cache]
    kv.appendToCache(cache, x, x, lens)
    want = on_cpu(kv.KeyValueCache(*before))
    oracle.append(want, x.cpu(), x.cpu(), [2, 0], None, None, None, "int8")
    assert torch.equal(cache.k.cpu().double(), want[0])
    q = r(2, 2, 3, 64)
    check(kv.AttentionOverCache(q, cache, lens), *expected(q, cache, lens))
    full = ints([4, 9])
    check(kv.AttentionOverCache(q, cache, full), *expected(q, cache, full))
    parents = ints([[-1, 0, 1]] * 2)
    check(kv.AttentionOverCache(q, cache, lens, parents), *expected(q, cache, lens, parents))


def test_empty_calls():
    kv = load("cache")
    cache = kv.newCache(2, 1, 4, 64)
    x = torch.zeros(2, 1, 0, 64, device="cuda")
    assert kv.appendToCache(cache, x, x, ints([0, 0]), q=x).shape == x.shape
    assert kv.AttentionOverCache(x, cache, ints([0, 0])).shape == x.shape
    none = kv.newCache(0, 1, 4, 64)
    y = torch.zeros(0, 1, 2, 64, device="cuda")
    assert kv.appendToCache(none, y, y, ints([])) is None and kv.AttentionOverCache(y, none, ints([])).shape == y.shape
    assert kv.readCache(none, ints([]), 3)[0].shape == (0, 1, 3, 64) and kv.keepDrafts(none, ints([]), torch.zeros(0, 2, dtype=torch.int32, device="cuda"), ints([])).shape == (0,)


def test_operators_refuse():
    kv, error, r = load("cache"), load("_lib").MarianHipError, maker(1)
    cache = kv.newCache(2, 2, 16, 64)
    k, lens = r(2, 2, 3, 64), ints([1, 2])
    q = r(2, 4, 3, 64)
    tree = ints([[-1, 0, 0]] * 2)
    bad = [lambda: kv.appendToCache(cache, k, k[:, :, :2], lens), lambda: kv.appendToCache(cache, k.half(), k, lens),
           lambda: kv.appendToCache(cache, k[:1], k[:1], lens), lambda: kv.appendToCache(cache, k, k, lens[:1]), lambda: kv.appendToCache(cache, k, k, lens.float()),
           lambda: kv.appendToCache(cache, k, k, lens, tree[:, :2]), lambda: kv.appendToCache(cache, k, k, lens, counts=lens[:1]),
           lambda: kv.appendToCache(cache, k, k, lens, q=q[:, :, :2]), lambda: kv.appendToCache(cache, k, k, lens, qOut=q),
           lambda: kv.appendToCache(cache, k, k, lens, rotary=kv.makeRotary(128)), lambda: kv.appendToCache(cache[:3], k, k, lens),
           lambda: kv.appendToCache(kv.KeyValueCache(cache.k, cache.v.view(torch.float8_e4m3fn), *cache[2:]), k, k, lens),
           lambda: kv.appendToCache(kv.KeyValueCache(cache.k, cache.k, *cache[2:]), k, k, lens),
           lambda: kv.appendToCache(kv.KeyValueCache(*(t[:, :, :8] for t in cache)), k, k, lens),
           lambda: kv.readCache(cache, lens, 2, torch.int8), lambda: kv.readCache(cache, lens, -1), lambda: kv.readCache(cache, lens[:1], 2),
           lambda: kv.AttentionOverCache(r(2, 3, 3, 64), cache, lens), lambda: kv.AttentionOverCache(q, cache, lens, scale=0.0),
           lambda: kv.AttentionOverCache(q, cache, lens, scale=-1.0), lambda: kv.AttentionOverCache(q.double(), cache, lens),
           lambda: kv.AttentionOverCache(q[..., :32], cache, lens), lambda: kv.AttentionOverCache(q, cache, lens.cpu()),
           lambda: kv.AttentionOverCache(q, cache, lens, out=q), lambda: kv.AttentionOverCache(q, cache, lens, out=q[:, :, :2]),
           lambda: kv.AttentionOverCache(r(2, 4, 65, 64), cache, lens, ints([[-1] * 65] * 2)),
           lambda: kv.keepDrafts(cache, lens, torch.zeros(2, 65, dtype=torch.int32, device="cuda"), lens), lambda: kv.keepDrafts(cache, lens, lens, lens),
           lambda: kv.keepDrafts(cache, lens, tree.float(), lens)]
    before = [t.clone() for t in cache]
    for i, call in enumerate(bad):
        with pytest.raises(error):
            say("refusal", i)
            call()
    assert all(same(a, b) for a, b in zip(cache, before))


def test_entries_far_apart():
    """Rows beyond 4 GB of a cache: written, read, attended to and moved"""
    kv, r = load("cache"), maker(2)
    S, H, cap, dk = 3, 16, 800000, 128
    cache = kv.newCache(S, H, cap, dk)
    lens = ints([5, 0, cap - 40])
    k, q = r(S, H, 33, dk), r(S, H, 33, dk)
    kv.appendToCache(cache, k, -k, lens)
    # (nothing before the new rows of the last sequence but zeros: its answer on the CPU needs the rows alone)
    got = kv.readCache(cache, lens, 33)[0][2]
    near = cache.k[2, :, cap - 40:cap - 7]
    assert torch.equal(got.cpu(), near.float().cpu() * cache.kScale[2, :, cap - 40:cap - 7, None].cpu()) and bool(near.abs().amax(-1).eq(127).all())
    moved = kv.keepDrafts(cache, lens, ints([[1, 32]] * S), ints([0, 1, 2]))
    assert moved.tolist() == [5, 1, cap - 38]
    assert torch.equal(kv.readCache(cache, lens, 2)[1][2], -got[:, [1, 32]])   # (codes of 0 have no sign)
    lens = ints([5, 0, 0])
    small = kv.KeyValueCache(*(t[2:, 15:, :64].contiguous() for t in cache))
    kv.appendToCache(small, k[2:, 15:], k[2:, 15:], lens[2:])
    kv.appendToCache(cache, k, k, lens)
    assert same(kv.AttentionOverCache(q, cache, lens)[2:, 15:], kv.AttentionOverCache(q, cache, lens)[2:, 15:])
    check(kv.AttentionOverCache(q, cache, lens)[2:, 15:], *expected(q[2:, 15:], small, lens[2:]))


# ---- accepted drafts ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("format", ["int8", "e4m3"])
@pytest.mark.parametrize("S,H,cap,dk,a", [(1, 1, 8, 16, 1), (4, 3, 100, 80, 9), (3, 2, 70, 256, 64), (5, 1, 40, 64, 0)])
def test_keep(format, S, H, cap, dk, a):
    kv, r = load("cache"), maker(a)
    cache = filled(r, S, H, cap, dk, format)
    before = [t.clone() for t in cache]
    lens = [(3, cap - 5, 0, -1, cap + 2)[s % 5] for s in range(S)]
    accepted = [(a, a + 4, a // 2, -2, a)[s % 5] for s in range(S)]
    g = torch.Generator().manual_seed(a)
    path = torch.randint(-1, 64, (S, a), generator=g)   # in any order, the same ones again, and ones that are not there
    got = kv.keepDrafts(cache, ints(lens), path.cuda(), ints(accepted))
    for s in range(S):
        first = oracle.clamp(lens[s], 0, cap)
        m = min(oracle.clamp(accepted[s], 0, a), cap - first)
        assert got[s] == first + m and got.dtype == torch.int32
        for t, b in zip(cache, before):
            want = b[s].clone()
            for j in range(m):
                if 0 <= path[s, j] < cap - first:
                    want[:, first + j] = b[s, :, first + int(path[s, j])]
            assert same(t[s], want)


# ---- together -------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,format", [(F32, "int8"), (BF16, "e4m3")])
def test_a_run_of_steps(dtype, format):
    """Prompts, drafted trees, their judgement and single tokens, against the same in 64 bits; then two hypotheses of one
    sequence by the framework's own state selection"""
    kv, ops, r = load("cache"), load("ops"), maker(21)
    S, H, G, dk, cap = 3, 2, 4, 64, 80
    rotary = kv.makeRotary(32, scaling="linear", factor=2.0)
    cache, want = kv.newCache(S, H, cap, dk, format), None
    want = on_cpu(cache)
    lens = ints([0, 0, 0])
    tree = ints([[-1, 0, 0, 1, 3, -1], [-1, -1, 1, 2, 2, 4], [-1, 0, 1, 2, 3, 4]])
    steps = [(23, None, ints([23, 7, 15])), (6, tree, None), (1, None, None), (6, tree, ints([6, 3, 0])), (1, None, None)]
    for n, parents, counts in steps:
        k, v = side_by_side(r, S, H, n, dk, dtype), side_by_side(r, S, H, n, dk, dtype)
        q = side_by_side(r, S, H * G, n, dk, dtype)
        near = oracle.append(want, k.cpu(), v.cpu(), lens.cpu(), oracle.cpu(parents), oracle.cpu(counts), rotary, format)
        turned = kv.appendToCache(cache, k, v, lens, parents, counts, rotary, q)
        kc, vc, ks, vs = on_cpu(cache)
        assert not ((kc != want[0]) & ~near).any() and torch.equal(vc, want[1]) and torch.equal(vs, want[3])
        want = [kc, vc, ks, vs]
        got = kv.AttentionOverCache(turned, cache, lens, parents, counts)
        check(got, *oracle.attention(turned.cpu(), kc, vc, ks, vs, lens.cpu(), oracle.cpu(parents), oracle.cpu(counts), dk ** -0.5))
        if parents is None:
            lens = lens + (n if counts is None else counts)
        else:   # the longest branches were right
            path, accepted = ints([[0, 1, 3, 4], [1, 2, 4, 5], [0, 1, 2, 3]]), ints([4, 1, 0])
            before = want
            old = lens.tolist()
            lens = kv.keepDrafts(cache, lens, path, accepted)
            want = [t.clone() for t in before]
            for s in range(S):
                for j in range(int(accepted[s])):
                    for t, b in zip(want, before):
                        t[s, :, old[s] + j] = b[s, :, old[s] + int(path[s, j])]
            assert all(torch.equal(a, b) for a, b in zip(on_cpu(cache), want)) and lens.tolist() == [o + int(m) for o, m in zip(old, accepted)]
    # beam search's selection: rows of the float32 views
    parents = ints([2, 0, 2])
    picked = []
    for t in cache:
        state = t.view(torch.int8).view(S, H, -1).view(F32) if t.element_size() == 1 else t.view(S, H, -1)
        out = torch.empty_like(state)
        ops.selectState(state, parents, out)
        picked.append(out.view(t.dtype).view(t.shape))
    assert all(same(p, t[[2, 0, 2]]) for p, t in zip(picked, cache))


def step_inputs(seed, S=5, H=2, G=4, n=6, dk=128, cap=3000, dtype=BF16):
    kv, r = load("cache"), maker(seed)
    cache = filled(r, S, H, cap, dk, "int8", 0.2)
    q, k, v = (side_by_side(r, S, h, n, dk, dtype) for h in (H * G, H, H))
    lens = ints([cap - n - 100 * s for s in range(S)])
    parents = ints([[-1, 0, 0, 1, 1, 2]] * S)
    rotary = kv.makeRotary(64)

    def step():
        turned = kv.appendToCache(cache, k, v, lens, parents, None, rotary, q)
        o = kv.AttentionOverCache(turned, cache, lens, parents)
        one = kv.AttentionOverCache(turned[:, :, :1], cache, lens)
        x = kv.rotaryPositions(o, lens, rotary)
        ks, vs = kv.readCache(cache, lens, n, dtype)
        return turned, o, one, x, ks, vs
    return step


def test_graphs_replay():
    """Recorded and replayed several times with eager work in between, and two graphs recorded on one stream replayed on two at once"""
    steps = [step_inputs(1), step_inputs(2)]
    want = [[t.clone() for t in step()] for step in steps]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for step in steps:
            step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for step in steps:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(step())
        graphs.append(g)
    others = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(4):
        for o in outs:
            for t in o:
                t.fill_(7.0)
        eager = steps[0]()
        assert all(same(a, b) for a, b in zip(eager, want[0]))
        torch.cuda.synchronize()
        for g, o in zip(graphs, others):
            with torch.cuda.stream(o):
                g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert all(same(a, b) for a, b in zip(o, w)), turn


def test_two_threads_with_a_stream_each():
    want, failed = {}, []
    for i in range(2):
        want[i] = [t.clone() for t in step_inputs(i + 5)()]
    torch.cuda.synchronize()

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                step = step_inputs(i + 5)
                for _ in range(30):
                    got = step()
                torch.cuda.current_stream().synchronize()
                assert all(same(a, b) for a, b in zip(got, want[i]))
        except BaseException as e:   # noqa: B902
            failed.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


# ---- calls at the edges -----------------------------------------------------------------------------------------
def test_rows_that_share_memory():
    """Expanded keys, values and queries are read as they are; expanded outputs, in place or not, are refused"""
    kv, error, r = load("cache"), load("_lib").MarianHipError, maker(3)
    S, H, G, n, dk = 3, 2, 4, 5, 64
    rotary = kv.makeRotary(dk)
    lens = ints([0, 3, 9])
    one = r(1, 1, n, dk)
    k, q = one.expand(S, H, n, dk), one.expand(S, H * G, n, dk)
    a, b = kv.newCache(S, H, 20, dk), kv.newCache(S, H, 20, dk)
    turned = kv.appendToCache(a, k, k, lens, rotary=rotary, q=q)
    again = kv.appendToCache(b, k.contiguous(), k.contiguous(), lens, rotary=rotary, q=q.contiguous())
    assert same(turned, again) and all(same(x, y) for x, y in zip(a, b))
    assert same(kv.AttentionOverCache(q, a, lens), kv.AttentionOverCache(q.contiguous(), a, lens))
    assert same(kv.rotaryPositions(q, lens, rotary), kv.rotaryPositions(q.contiguous(), lens, rotary))
    before = [t.clone() for t in a]
    for call in (lambda: kv.rotaryPositions(q, lens, rotary, out=q), lambda: kv.appendToCache(a, k.contiguous(), k.contiguous(), lens, rotary=rotary, q=q, qOut=q),
                 lambda: kv.AttentionOverCache(turned, a, lens, out=r(S, 1, n, dk).expand(S, H * G, n, dk))):
        with pytest.raises(error):
            call()
    assert all(same(x, y) for x, y in zip(a, before))


@pytest.mark.parametrize("interleaved", [False, True])
def test_in_place(interleaved):
    kv, r = load("cache"), maker(4)
    S, H, n, dk = 2, 3, 9, 80
    rotary = kv.makeRotary(48, interleaved=interleaved)
    lens = ints([5, 1000])
    for lay in (lambda: r(S, H, n, dk), lambda: side_by_side(r, S, H, n, dk, BF16)):
        x = lay()
        want = kv.rotaryPositions(x, lens, rotary)
        cache, other = kv.newCache(S, H, 1100, dk), kv.newCache(S, H, 1100, dk)
        k = x.clone()
        q = kv.appendToCache(cache, k, k, lens, rotary=rotary, q=x)
        y = x.clone()
        assert kv.rotaryPositions(y, lens, rotary, out=y) is not None and same(y, want)
        y = x.clone()
        kv.appendToCache(other, k, k, lens, rotary=rotary, q=y, qOut=y)
        assert same(y, q) and all(same(a, b) for a, b in zip(cache, other))


def test_positions_at_the_ends_of_32_bits():
    """Row i stands at positions[s] + i also where that passes 2^31 - 1; lengths of 64 bits are beyond any capacity"""
    kv, r = load("cache"), maker(5)
    x = r(2, 1, 4, 64)
    rotary = kv.makeRotary(64)
    first = [2 ** 31 - 2, -2 ** 31]
    got = kv.rotaryPositions(x, ints(first), rotary).cpu()
    turns = [int(t) % 2 ** 64 for t in rotary.turns.cpu()]
    for s in range(2):
        for i in range(4):
            for p in range(32):
                angle = 2 * math.pi * ((first[s] + i) * turns[p] % 2 ** 64) / 2 ** 64
                a, b = float(x[s, 0, i, p]), float(x[s, 0, i, p + 32])
                size = abs(a) + abs(b)
                # an angle in float32, up to a half turn: 2^-24 of it; sine and cosine within 2 steps; two products and a sum
                bound = size * (math.pi * 2 ** -23 + 6 * 2 ** -24)
                assert abs(float(got[s, 0, i, p]) - (a * math.cos(angle) - b * math.sin(angle))) <= bound
                assert abs(float(got[s, 0, i, p + 32]) - (a * math.sin(angle) + b * math.cos(angle))) <= bound
    cache = filled(r, 2, 1, 10, 64, "int8")
    far = torch.tensor([2 ** 32 + 3, -2 ** 32], device="cuda")
    near = ints([10, 0])
    q = r(2, 1, 1, 64)
    assert same(kv.AttentionOverCache(q, cache, far), kv.AttentionOverCache(q, cache, near))
    assert kv.keepDrafts(cache, far, ints([[0], [0]]), ints([1, 1])).tolist() == [10, 1]


def test_lengths_that_grow_on_one_stream_and_codes_from_elsewhere():
    """Calls of all sizes after each other, the workspace growing on the way and serving the smaller ones again; e4m3's NaN codes
    and int8's -128 are taken by their bits, alike by attention and reading"""
    kv, r = load("cache"), maker(6)
    for dtype in (F32, BF16):
        for n, H, cap in ((1, 8, 3000), (40, 2, 5000), (1, 8, 3000), (130, 1, 900), (64, 8, 700), (1, 1, 9000)):
            cache = filled(r, 2, H, cap, 64, "int8")
            q, lens = r(2, 2 * H, n, 64).to(dtype), ints([cap - n, cap // 3])
            check(kv.AttentionOverCache(q, cache, lens), *expected(q, cache, lens))
    for format, bits, value in (("e4m3", 0x7f, 480.0), ("e4m3", 0xff, -480.0), ("int8", 0x80, -128.0)):
        cache = kv.newCache(1, 1, 4, 64, format)
        for t in cache[:2]:
            t.view(torch.uint8).fill_(bits)
        for t in cache[2:]:
            t.fill_(0.5)
        assert all((x == value / 2).all() for x in kv.readCache(cache, ints([0]), 4))
        # (the sum is divided by through its reciprocal, and weights are exponentials: not exact even here, but within the oracle's
        # bound, which counts both)
        q, codes, scales = torch.ones(1, 1, 1, 64), torch.full((1, 1, 4, 64), value, dtype=torch.float64), torch.full((1, 1, 4), 0.5)
        got = kv.AttentionOverCache(q.cuda(), cache, ints([3]))
        check(got, *oracle.attention(q, codes, codes, scales, scales, torch.tensor([3]), None, None, 0.125))


@pytest.mark.parametrize("S,H,G,cap", [(32, 32, 8, 64), (32, 32, 8, 400), (32, 32, 1, 64), (16, 16, 24, 64), (8, 16, 40, 64), (4, 8, 150, 64)])
def test_every_weight_of_float32(S, H, G, cap):
    """Values that are a row of the identity each show the weights one by one: all within what their scores may be off (some 2^-13 here),
    none short of its second float16 (2^-11 of it)"""
    kv, r = load("cache"), maker(G + cap)
    cache = kv.newCache(S, H, cap, 64)
    k, v = r(S, H, 64, 64), torch.eye(64, device="cuda") * torch.exp(0.3 * r(S, H, 64, 1))   # (scales of their own)
    kv.appendToCache(cache, k, v, ints([0] * S))
    q = r(S, H * G, 1, 64)
    lens = ints([63] * S)
    small = kv.KeyValueCache(*(t[:, :, :64] for t in cache))
    want, tol = expected(q, small, lens)
    assert (tol[want > 1e-3] < want[want > 1e-3] * 2.0 ** -12).all()
    check(kv.AttentionOverCache(q, cache, lens), want, tol)


@pytest.mark.parametrize("S,H,G,n,dk", [(3, 2, 2, 1500, 64), (1, 8, 4, 1001, 128), (40, 4, 1, 67, 256), (70, 16, 1, 63, 64)])
def test_append_of_many_tokens(S, H, G, n, dk):
    """Alike whether a workgroup takes four tokens or one: all at once, and in pieces"""
    kv, r = load("cache"), maker(n)
    rotary = kv.makeRotary(dk, base=50000.0)
    whole, pieces = kv.newCache(S, H, n + 9, dk, "e4m3"), kv.newCache(S, H, n + 9, dk, "e4m3")
    k, v, q = side_by_side(r, S, H, n, dk, BF16), side_by_side(r, S, H, n, dk, BF16), side_by_side(r, S, H * G, n, dk, BF16)
    lens = [s % 7 for s in range(S)]
    counts = [n - (s * 5) % 11 for s in range(S)]
    turned = kv.appendToCache(whole, k, v, ints(lens), None, ints(counts), rotary, q)
    for i in range(0, n, 16):
        m = min(16, n - i)
        part = kv.appendToCache(pieces, k[:, :, i:i + m], v[:, :, i:i + m], ints([x + i for x in lens]), None, ints([c - i for c in counts]), rotary, q[:, :, i:i + m])
        assert same(part, turned[:, :, i:i + m])
    assert all(same(a, b) for a, b in zip(whole, pieces))

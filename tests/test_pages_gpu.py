"""The cache in pages and the attention over it on the GPU, against the same written out in 64 bits on the CPU (pages_oracle.py, which says how
far results may be)."""
import random
import threading

import pytest
import torch

import pages_oracle as oracle
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
    bad = ~((got - want).abs() <= tol) & ~(torch.isnan(got) & torch.isnan(want)) & ~(torch.isinf(got) & (got == want))
    assert not bad.any(), "%d of %d off, first at %s: %r, %r +- %r" % (
        bad.sum(), bad.numel(), bad.nonzero()[0].tolist(), got[bad][0].item(), want[bad][0].item(), tol[bad][0].item())


def dealt(seed, lens, page, row, pages):
    """a table in which every sequence has the pages that its length needs, in no order"""
    order = list(range(pages))
    random.Random(seed).shuffle(order)
    table = [[-1] * row for _ in lens]
    for s, n in enumerate(lens):
        for j in range(min(row, -(-n // page))):
            table[s][j] = order.pop()
    return table


def poisoned(r, table, lens, page, pages, heads, dk, dtype):
    """keys and values ~N(0, 1) at the positions that sequences have, NaN everywhere else"""
    kv = load("pages").newPagedCache(pages, heads, page, dk, dtype)
    k, v = kv
    k.fill_(float("nan"))
    v.fill_(float("nan"))
    for s, n in enumerate(lens):
        for j, p in enumerate(table[s]):
            here = min(page, n - j * page)
            if here > 0 and 0 <= p < pages:
                k[p, :, :here] = r(heads, here, dk).to(dtype)
                v[p, :, :here] = r(heads, here, dk).to(dtype)
    return kv


def expected(q, kv, table, lens, counts=None, scale=None):
    return oracle.attention(q.cpu(), kv.k.cpu(), kv.v.cpu(), table.cpu(), lens, counts, scale or q.shape[-1] ** -0.5)


# ---- attention -------------------------------------------------------------------------------------------
SHAPES = [   # sequences, heads of keys, query heads to each, new tokens, dk, positions of a page, lengths
    (1, 1, 1, 1, 16, 8, [0]), (1, 1, 1, 1, 64, 16, [1]), (3, 2, 1, 1, 64, 16, [0, 31, 32]), (2, 3, 5, 1, 80, 24, [127, 128]),
    (4, 2, 4, 1, 128, 16, [129, 7, 0, 300]), (2, 2, 8, 1, 96, 40, [511, 513]), (2, 1, 16, 1, 128, 256, [257, 1000]), (1, 2, 17, 1, 64, 8, [700]),
    (2, 2, 1, 1, 256, 32, [33, 260]), (1, 1, 32, 1, 256, 64, [1030]), (1, 1, 4, 1, 128, 4096, [5000]), (1, 2, 1, 1, 64, 16, [4999]),
    (2, 2, 2, 2, 64, 16, [15, 0]), (3, 1, 4, 7, 128, 16, [120, 121, 640]), (2, 2, 8, 7, 128, 8, [1000, 9]), (2, 1, 3, 21, 80, 48, [60, 333]),
    (1, 2, 4, 33, 64, 32, [700]), (2, 1, 2, 130, 128, 16, [0, 77]), (1, 1, 1, 64, 256, 16, [200]), (2, 2, 1, 16, 112, 56, [40, 1500]),
    (1, 1, 8, 40, 256, 128, [99])]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("S,heads,group,n,dk,page,lens", SHAPES)
def test_attention(dtype, S, heads, group, n, dk, page, lens):
    pages, r = load("pages"), maker(S + n + dk)
    row = -(-(max(lens) + n) // page) + 1
    table = dealt(n, [l + n for l in lens], page, row, S * row + 3)
    kv = poisoned(r, table, [l + n for l in lens], page, S * row + 3, heads, dk, dtype)
    q = side_by_side(r, S, heads * group, n, dk, dtype)
    table = ints(table)
    want, tol = expected(q, kv, table, lens)
    say("attention", dtype, S, heads, group, n, dk, page, lens)
    got = pages.AttentionOverPages(q, kv, table, ints(lens))
    assert got.shape == q.shape and got.dtype == dtype
    check(got, want, tol)
    # counts; lens as int64; queries head by head; into a part of another tensor; another scale; a table that is a part of a wider one
    counts = [(n + s) // 2 for s in range(S)]
    some, some_tol = expected(q, kv, table, lens, counts)
    got = pages.AttentionOverPages(q, kv, table, ints(lens).long(), ints(counts))
    check(got, some, some_tol)
    for s in range(S):
        assert not got[s, :, counts[s]:].any()
    out = torch.full((S, heads * group, n, 2 * dk), 7.0, dtype=dtype, device="cuda")
    assert pages.AttentionOverPages(q.contiguous(), kv, table, ints(lens), out=out[..., dk:]).data_ptr() == out[..., dk:].data_ptr()
    check(out[..., dk:], want, tol)
    assert (out[..., :dk] == 7.0).all()
    want, tol = expected(q, kv, table, lens, scale=0.5)
    wide = torch.full((S, row + 5), -1, dtype=torch.int32, device="cuda")
    wide[:, :row] = table
    check(pages.AttentionOverPages(q, kv, wide, ints(lens), scale=0.5), want, tol)
    check(pages.AttentionOverPages(q, kv, wide[:, :row], ints(lens), scale=0.5), want, tol)


FORMS = [(dk, group, n, seqs) for dk in (64, 48, 128, 80, 256, 144) for group, n in ((1, 1), (5, 4), (8, 7), (16, 6)) for seqs in (3, 1030)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dk,group,n,S", FORMS)
def test_every_form_of_the_attention(dtype, dk, group, n, S):
    """(tests/test_pages.py asks the plan whether these launch them all); few sequences with long contexts in several parts, or many of one wave"""
    pages, r = load("pages"), maker(dk + n)
    heads, page = (2, 32) if S < 100 else (4, 8)
    lens = [(700, 0, 1400)[s % 3] if S < 100 else s % 12 for s in range(S)]
    row = 60 if S < 100 else 5
    table = dealt(7, [l + n for l in lens], page, row, S * row)
    kv = poisoned(r, table, [l + n for l in lens], page, S * row, heads, dk, dtype) if S < 100 else None
    if kv is None:   # (written at once: NaN behind the last token of every page)
        kv = pages.newPagedCache(S * row, heads, page, dk, dtype)
        kv.k.fill_(float("nan"))
        kv.v.fill_(float("nan"))
        longest = max(lens) + n
        slots = torch.full((S, longest), -1, dtype=torch.int32)
        for s in range(S):
            for i in range(lens[s] + n):
                slots[s, i] = table[s][i // page] * page + i % page
        pages.writePages(kv, side_by_side(r, S, heads, longest, dk, dtype), side_by_side(r, S, heads, longest, dk, dtype), slots.cuda())
    q = side_by_side(r, S, heads * group, n, dk, dtype)
    got = pages.AttentionOverPages(q, kv, ints(table), ints(lens))
    some = list(range(0, S, 1 if S < 100 else 29))   # (the oracle takes its time)
    check(got[some], *expected(q[some], kv, ints(table)[some], [lens[s] for s in some]))
    assert torch.isfinite(got).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_attention_of_many_short_sequences(dtype):
    """(a workgroup of one wave to each)"""
    pages, r = load("pages"), maker(3)
    S, heads, group, dk, page = 300, 16, 2, 64, 16
    lens = [(7 * s) % 50 for s in range(S)]
    table = dealt(1, [l + 1 for l in lens], page, 4, S * 4)
    kv = poisoned(r, table, [l + 1 for l in lens], page, S * 4, heads, dk, dtype)
    q = side_by_side(r, S, heads * group, 1, dk, dtype)
    check(pages.AttentionOverPages(q, kv, ints(table), ints(lens)), *expected(q, kv, ints(table), lens))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_attention_over_lengths_that_differ(dtype):
    """(long ones in several parts, beside short ones that stay whole)"""
    pages, r = load("pages"), maker(4)
    S, heads, group, dk, page = 5, 2, 4, 128, 32
    lens = [9000, 3, 0, 2600, 640]
    row = 290
    table = dealt(2, [l + 3 for l in lens], page, row, 500)
    kv = poisoned(r, table, [l + 3 for l in lens], page, 500, heads, dk, dtype)
    q = side_by_side(r, S, heads * group, 3, dk, dtype)
    got = pages.AttentionOverPages(q, kv, ints(table), ints(lens))
    check(got, *expected(q, kv, ints(table), lens))
    for _ in range(3):
        assert same(pages.AttentionOverPages(q, kv, ints(table), ints(lens)), got)   # (whoever comes last)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_pages_that_are_none_are_not_seen(dtype):
    pages, r = load("pages"), maker(5)
    S, heads, group, dk, page = 4, 2, 2, 64, 16
    lens = [100, 100, 40, 200]
    table = dealt(3, [l + 2 for l in lens], page, 8, 40)   # (the last one's row is too short)
    table[0][2], table[0][5] = -1, 40       # none, and past the last
    table[1][0] = -2 ** 31
    table[1][6] = 2 ** 31 - 1               # the new tokens' own page
    table[2] = [-1] * 8                     # nothing at all
    kv = poisoned(r, table, [l + 2 for l in lens], page, 40, heads, dk, dtype)
    q = side_by_side(r, S, heads * group, 2, dk, dtype)
    want, tol = expected(q, kv, ints(table), lens)
    assert not want[2].any() and torch.isfinite(want).all()
    check(pages.AttentionOverPages(q, kv, ints(table), ints(lens)), want, tol)
    # lengths outside the row
    got = pages.AttentionOverPages(q, kv, ints(table), ints([-5, 2 ** 31 - 1, 0, 128]))
    want, tol = expected(q, kv, ints(table), [0, 128, 0, 128])
    check(got, want, tol)
    # sequences that share all they have
    shared = ints([table[0]] * 4)
    got = pages.AttentionOverPages(q[:1].expand(4, -1, -1, -1).contiguous(), kv, shared, ints([100] * 4))
    assert all(same(got[i], got[0]) for i in range(4))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dk", [64, 128, 256])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("group,n", [(4, 5), (8, 7), (8, 20)])
def test_what_a_token_does_not_see_is_not_in_its_result(dtype, dk, bad, group, n):
    """A chain of tokens, the fourth of which holds an infinity or NaN in some places: the first three are as without it"""
    pages, r = load("pages"), maker(6)
    heads, page = 2, 8
    for past in (0, 26, 60, 130):
        row = 20
        table = dealt(4, [past + n], page, row, row)
        kv = poisoned(r, table, [past + n], page, row, heads, dk, dtype)
        q = side_by_side(r, 1, heads * group, n, dk, dtype)
        clean = pages.AttentionOverPages(q, kv, ints(table), ints([past]))
        p, at = table[0][(past + 3) // page], (past + 3) % page
        kv.v[p, 0, at, 5] = bad
        kv.v[p, 1, at, dk - 1] = bad
        got = pages.AttentionOverPages(q, kv, ints(table), ints([past]))
        assert same(got[:, :, :3], clean[:, :, :3])
        want, tol = expected(q, kv, ints(table), [past])
        assert not torch.isfinite(want[0, :, 3:]).all()
        check(got, want, torch.where(torch.isfinite(want), tol, torch.zeros_like(tol)))
        if past:   # ... and a settled one, that all see
            kv.v[table[0][past // 2 // page], 1, past // 2 % page, 7] = bad
            got = pages.AttentionOverPages(q, kv, ints(table), ints([past]))
            want, tol = expected(q, kv, ints(table), [past])
            assert not torch.isfinite(want[0, group:, :, 7]).any()
            check(got, want, torch.where(torch.isfinite(want), tol, torch.zeros_like(tol)))
            clean = got
        kv.k[p, :, at] = bad
        got = pages.AttentionOverPages(q, kv, ints(table), ints([past]))
        assert same(got[:, :, :3].nan_to_num(), clean[:, :, :3].nan_to_num()) and torch.isnan(got[0, :group, 4:, 5]).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dk", [64, 128, 256])
@pytest.mark.parametrize("group,n", [(4, 1), (8, 4), (8, 7), (8, 16)])
def test_infinities_in_long_sequences(dtype, dk, group, n):
    """Settled positions of every turn's both halves, in one part of a sequence or another: an infinity that all see is their result, NaN
    where a later position has one of the other sign or NaN; all else is as without"""
    pages, r = load("pages"), maker(9)
    heads, page, past = 2, 16, 2500
    row = -(-(past + n) // page)
    table = dealt(6, [past + n], page, row, row)
    kv = poisoned(r, table, [past + n], page, row, heads, dk, dtype)
    q = side_by_side(r, 1, heads * group, n, dk, dtype)
    inf = float("inf")
    for at, d, x in ((3, 0, inf), (40, 1, -inf), (700, 2, inf), (1333, 3, -inf), (64, 4, inf), (2100, 4, -inf), (95, 5, inf), (2499, 5, float("nan"))):
        kv.v[table[0][at // page], 1, at % page, d] = x
    got = pages.AttentionOverPages(q, kv, ints(table), ints([past]))
    want, tol = expected(q, kv, ints(table), [past])
    assert torch.isinf(want[0, group:, :, :4]).all() and torch.isnan(want[0, group:, :, 4:6]).all() and torch.isfinite(want[0, :group]).all()
    check(got, want, torch.where(torch.isfinite(want), tol, torch.zeros_like(tol)))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("share", [1.0, 0.99])
def test_values_next_to_the_largest(dtype, share):
    """Results are means of values, and stay in range where what they may be off by does: the mean of values that are all the largest number M
    is M (1 + d), |d| <= tol, and every number above M is infinity, so for share 1 an infinity is as near as any other result"""
    pages, r = load("pages"), maker(7)
    top = torch.finfo(dtype).max
    for lens in ([3000], [40000]):
        row = -(-(lens[0] + 1) // 64)
        table = dealt(5, [lens[0] + 1], 64, row, row)
        kv = poisoned(r, table, [lens[0] + 1], 64, row, 1, 64, dtype)
        kv.v.fill_(top * share)
        q = side_by_side(r, 1, 4, 1, 64, dtype) * 30
        got = pages.AttentionOverPages(q, kv, ints(table), ints(lens)).double()
        tol = 2 * oracle.HALF[dtype] + (lens[0] + 8) * 2.0 ** -23
        want = kv.v[0, 0, 0, 0].double()
        assert (((got / want - 1).abs() <= tol) | ((got == float("inf")) & (want * (1 + tol) > top))).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_cache_past_32_bits(dtype):
    """Pages whose values lie more than 2^32 bytes, and 2^31 values, behind the first"""
    pages, r = load("pages"), maker(8)
    heads, page, dk = 8, 64, 128
    count = (1 << 31) // (heads * page * dk) + 300
    kv = pages.PagedCache(*(torch.empty(count, heads, page, dk, dtype=dtype, device="cuda") for _ in "kv"))
    lens = [200, 500]
    table = [[count - 1 - 3 * j for j in range(8)], [count - 2 - 3 * j for j in range(8)]]
    slots = torch.full((2, 504), -1, dtype=torch.int32)
    for s in range(2):
        for i in range(lens[s] + 1):
            slots[s, i] = table[s][i // page] * page + i % page
    k, v = side_by_side(r, 2, heads, 504, dk, dtype), side_by_side(r, 2, heads, 504, dk, dtype)
    pages.writePages(kv, k, v, slots.cuda())
    q = side_by_side(r, 2, heads, 1, dk, dtype)
    got = pages.AttentionOverPages(q, kv, ints(table), ints(lens))
    first = 1 << 62
    for s in range(2):
        first = min(first, min(table[s]))
    small = pages.PagedCache(kv.k[first:].clone(), kv.v[first:].clone())
    for s in range(2):
        assert same(small.k[table[s][0] - first], k[s, :, :page]) and same(small.v[table[s][1] - first], v[s, :, page:2 * page])
    check(got, *expected(q, small, ints(table) - first, lens))


# ---- tables ------------------------------------------------------------------------------------------------
def as_lists(tables):
    return [t.tolist() for t in tables]


@pytest.mark.parametrize("S,row,pages,page,n", [(1, 1, 1, 8, 1), (6, 9, 40, 16, 1), (37, 12, 200, 24, 5), (1000, 6, 3000, 8, 3), (1025, 5, 2500, 16, 9),
                                                (5000, 4, 9000, 8, 2), (64, 140, 5000, 16, 2001), (300, 70, 9000, 64, 4000)])
def test_tables(S, row, pages, page, n):
    """Rounds of reserving and trimming, with counts and without, until the pages run out and beyond; every table as the oracle has it"""
    P, rng = load("pages"), random.Random(S)
    tables = P.newPageTables(S, row, pages)
    mirror = as_lists(tables)
    lens = [0] * S
    say("tables", S, row, pages, page, n)
    for turn in range(6):
        counts = [rng.randint(0, n) for _ in range(S)] if turn % 2 else None
        slots = P.reservePages(tables, ints(lens), n, page, None if counts is None else ints(counts))
        want = oracle.reserve(*mirror, lens, n, page, counts)
        assert slots.tolist() == want and as_lists(tables) == mirror, turn
        for s in range(S):   # some go on, some have some of their drafts refused, some are done
            m = n if counts is None else counts[s]
            room = all(x >= 0 for x in want[s][:m])
            lens[s] = 0 if rng.random() < 0.2 else lens[s] + rng.randint(0, m) if room else lens[s]
        P.trimPages(tables, ints(lens).long(), page)
        oracle.trim(*mirror, lens, page)
        assert as_lists(tables) == mirror, turn
    P.trimPages(tables, ints([0] * S), page)
    assert tables.freeCount.item() == pages and sorted(tables.free.tolist()) == list(range(pages)) and (tables.table == -1).all()


def test_tables_that_hold_anything():
    """Counts out of range are taken as the nearer end, negative lengths as none; nothing is written outside the tables"""
    P = load("pages")
    for seed in range(8):
        rng = random.Random(seed)
        S, row, pages, page, n = 20, 5, 30, 8, 11
        mirror = [[[rng.choice([-7, 3, 29, 30, 2 ** 31 - 1]) for _ in range(row)] for _ in range(S)],
                  [rng.choice([-3, 0, 2, 5, 9, 2 ** 31 - 1]) for _ in range(S)], [rng.choice([-1, 5, 30, 1000]) for _ in range(pages)],
                  [rng.choice([-4, 7, 30, 99])]]
        lens = [rng.choice([-9, 0, 3, 17, 39, 41, 2 ** 31 - 1]) for _ in range(S)]
        counts = [rng.choice([-1, 0, 3, 11, 50]) for _ in range(S)]
        guard = [torch.full((t.numel() + 64,), 77, dtype=torch.int32, device="cuda") for t in (ints(x) for x in mirror)]
        parts = [g[32:-32].view(ints(x).shape).copy_(ints(x)) for g, x in zip(guard, mirror)]
        tables = P.PageTables(*parts)
        assert P.reservePages(tables, ints(lens), n, page, ints(counts)).tolist() == oracle.reserve(*mirror, lens, n, page, counts), seed
        assert as_lists(tables) == mirror, seed
        P.trimPages(tables, ints(lens), page)
        oracle.trim(*mirror, lens, page)
        assert as_lists(tables) == mirror, seed
        assert all((g[:32] == 77).all() and (g[-32:] == 77).all() for g in guard)


def test_nothing_to_deal():
    P = load("pages")
    tables = P.newPageTables(3, 2, 4)
    assert P.reservePages(tables, ints([0, 0, 0]), 0, 8).shape == (3, 0)
    kv, none = P.newPagedCache(4, 2, 8, 64), torch.zeros(3, 2, 0, 64, device="cuda")
    P.writePages(kv, none, none, P.reservePages(tables, ints([0, 0, 0]), 0, 8))
    assert P.AttentionOverPages(none, kv, tables.table, ints([0, 0, 0])).shape == (3, 2, 0, 64)
    empty = P.newPageTables(0, 2, 4)
    assert P.reservePages(empty, ints([]), 5, 8).shape == (0, 5)
    P.trimPages(empty, ints([]), 8)
    assert P.AttentionOverPages(torch.zeros(0, 4, 1, 64, device="cuda"), P.newPagedCache(4, 2, 8, 64), empty.table, ints([])).shape == (0, 4, 1, 64)
    error = load("_lib").MarianHipError
    for call in (lambda: P.reservePages(tables, ints([0, 0]), 1, 8), lambda: P.reservePages(tables, ints([0, 0, 0]), 1, 12),
                 lambda: P.reservePages(tables, torch.zeros(3, device="cuda"), 1, 8), lambda: P.reservePages(tables, ints([0, 0, 0]), -1, 8),
                 lambda: P.reservePages(tables._replace(table=tables.table.long()), ints([0, 0, 0]), 1, 8),
                 lambda: P.reservePages(tables._replace(held=tables.free[:3]), ints([0, 0, 0]), 1, 8), lambda: P.trimPages(tables, ints([0] * 4), 8)):
        with pytest.raises(error):
            call()


# ---- writing -----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("S,heads,n,dk,page", [(1, 1, 1, 16, 8), (3, 2, 5, 80, 24), (2, 8, 33, 128, 16), (64, 4, 1, 64, 32), (1, 3, 700, 256, 4096)])
def test_writing(dtype, S, heads, n, dk, page):
    P, r, rng = load("pages"), maker(S + n), random.Random(n)
    pages = -(-S * n // page) + 2
    kv = P.newPagedCache(pages, heads, page, dk, dtype)
    kv.k.fill_(7)
    kv.v.fill_(8)
    places = rng.sample(range(pages * page), S * n)
    slots = [[places[s * n + i] if rng.random() < 0.9 else rng.choice([-1, -2 ** 31, pages * page, 2 ** 31 - 1]) for i in range(n)] for s in range(S)]
    k, v = side_by_side(r, S, heads, n, dk, dtype), side_by_side(r, S, heads, n, dk, dtype)
    want = [t.cpu() for t in kv]
    for s in range(S):
        for i, slot in enumerate(slots[s]):
            if 0 <= slot < pages * page:
                want[0][slot // page, :, slot % page] = k[s, :, i].cpu()
                want[1][slot // page, :, slot % page] = v[s, :, i].cpu()
    P.writePages(kv, k, v, ints(slots))
    assert same(kv.k.cpu(), want[0]) and same(kv.v.cpu(), want[1])
    # head by head, slots as int64, a value that all heads share, rows that have to be copied first
    P.writePages(kv, k.contiguous(), v[:, :1].expand(-1, heads, -1, -1), ints(slots).long())
    odd = torch.zeros(S * heads * n * dk + 1, dtype=dtype, device="cuda")[1:].view(S, heads, n, dk).copy_(k)
    for s in range(S):
        for i, slot in enumerate(slots[s]):
            if 0 <= slot < pages * page:
                want[1][slot // page, :, slot % page] = v[s, :1, i].cpu()
    assert same(kv.k.cpu(), want[0]) and same(kv.v.cpu(), want[1])
    P.writePages(kv, odd, v, ints(slots))
    assert same(kv.k.cpu(), want[0])
    error = load("_lib").MarianHipError
    for call in (lambda: P.writePages(kv, k[:, :, :, :16 if dk > 16 else 8], v, ints(slots)), lambda: P.writePages(kv, k.double(), v, ints(slots)),
                 lambda: P.writePages(kv, k, v, ints(slots)[:, :0]), lambda: P.writePages((kv.k, kv.v[:1]), k, v, ints(slots))):
        with pytest.raises(error):
            call()


# ---- as they are used ----------------------------------------------------------------------------------------
def test_attention_refusals():
    P, r, error = load("pages"), maker(1), load("_lib").MarianHipError
    kv = P.newPagedCache(6, 2, 16, 64, F16)
    q, table, lens = side_by_side(r, 2, 4, 1, 64, F16), ints([[0, 1], [2, 3]]), ints([3, 20])
    P.AttentionOverPages(q, kv, table, lens)
    for call in (lambda: P.AttentionOverPages(q.float(), kv, table, lens), lambda: P.AttentionOverPages(q[:, :3], kv, table, lens),
                 lambda: P.AttentionOverPages(q, kv, table[:1], lens), lambda: P.AttentionOverPages(q, kv, table, lens[:1]),
                 lambda: P.AttentionOverPages(q, kv, table.float(), lens), lambda: P.AttentionOverPages(q, kv, table, lens, scale=-1.0),
                 lambda: P.AttentionOverPages(q[..., :48], kv, table, lens), lambda: P.AttentionOverPages(q, kv, table, lens, out=q),
                 lambda: P.AttentionOverPages(q, kv, table, lens, out=kv.k[:2, :, :2].reshape(2, 4, 1, 64).expand(2, 4, 1, 64)[:, :, :, :32]),
                 lambda: P.AttentionOverPages(q, (kv.k.transpose(1, 2), kv.v.transpose(1, 2)), table, lens)):
        with pytest.raises(error):
            call()


def decode(P, kv_ops, caches, tables, project, steps, S, page, n, device="cuda"):
    """`steps` steps of n tokens of S sequences over all caches; returns what every layer gave"""
    outs, lens = [], torch.zeros(S, dtype=torch.int32, device=device)
    for step in range(steps):
        slots = P.reservePages(tables, lens, n, page)
        for layer, kv in enumerate(caches):
            q, k, v = project(step, layer)
            P.writePages(kv, k, v, slots)
            outs.append(P.AttentionOverPages(q, kv, tables.table, lens))
        kept = torch.full((S,), n, dtype=torch.int32, device=device) - torch.arange(S, device=device, dtype=torch.int32) % n
        lens = lens + kept.to(torch.int32)
        P.trimPages(tables, lens, page)
    return outs, lens


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_steps_of_a_decoder_with_refused_drafts(dtype):
    """Pages reserved, written, read and given back over several steps of two layers: every result is that of the plain formula over the tokens
    that were kept"""
    P, kv_ops, r = load("pages"), load("cache"), maker(9)
    S, heads, group, dk, page, n, steps = 3, 2, 2, 64, 8, 5, 7
    caches = [P.newPagedCache(30, heads, page, dk, dtype) for _ in "ab"]
    for kv in caches:
        kv.k.fill_(float("nan"))
        kv.v.fill_(float("nan"))
    tables = P.newPageTables(S, 8, 30)
    made = {(t, l): tuple(side_by_side(r, S, h, n, dk, dtype) for h in (heads * group, heads, heads)) for t in range(steps) for l in range(2)}
    outs, lens = decode(P, kv_ops, caches, tables, lambda t, l: made[t, l], steps, S, page, n)
    assert tables.held.tolist() == [-(-x // page) for x in lens.tolist()]
    for layer in range(2):
        for s in range(S):
            k = torch.zeros(heads, 0, dk, dtype=dtype)
            v = k
            for t in range(steps):
                q, kn, vn = (x[s:s + 1].cpu() for x in made[t, layer])
                past = k.shape[1]
                k, v = torch.cat((k, kn[0]), 1), torch.cat((v, vn[0]), 1)
                flat = [torch.zeros(1, heads, page * (-(-(past + n) // page)), dk, dtype=dtype) for _ in "kv"]
                flat[0][0, :, :past + n], flat[1][0, :, :past + n] = k, v
                pool = [x[0].view(heads, -1, page, dk).transpose(0, 1).contiguous() for x in flat]
                want, tol = oracle.attention(q, pool[0], pool[1], torch.arange(pool[0].shape[0])[None], [past], None, dk ** -0.5)
                check(outs[2 * t + layer][s:s + 1], want, tol)
                k, v = k[:, :past + n - s % n], v[:, :past + n - s % n]


def test_a_recorded_step_is_replayed():
    """Two graphs of the same step on the same tables, replayed in turn with eager steps between them: all as the eager ones"""
    P, kv_ops, r = load("pages"), load("cache"), maker(10)
    S, heads, group, dk, page, n = 4, 2, 4, 128, 16, 3
    kept = ints([1, 2, 3, 1])

    def fresh():
        return P.newPagedCache(60, heads, page, dk, BF16), P.newPageTables(S, 12, 60), torch.zeros(S, dtype=torch.int32, device="cuda")

    def step(state, q, k, v):
        kv, tables, lens = state
        slots = P.reservePages(tables, lens, n, page)
        P.writePages(kv, k, v, slots)
        out = P.AttentionOverPages(q, kv, tables.table, lens)
        lens += kept
        P.trimPages(tables, lens, page)
        return out, slots
    turns = [tuple(side_by_side(r, S, h, n, dk, BF16) for h in (heads * group, heads, heads)) for _ in range(9)]
    state = fresh()
    want = [tuple(x.clone() for x in step(state, *t)) for t in turns]
    end = [t.clone() for t in (*state[0], *state[1], state[2])]

    state = fresh()
    fixed = [torch.empty_like(x) for x in turns[0]]
    scratch = fresh()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(scratch, *turns[0])   # (before it is recorded)
    torch.cuda.current_stream().wait_stream(stream)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(state, *fixed)
        graphs.append((g, out))
    for i, t in enumerate(turns):
        for a, b in zip(fixed, t):
            a.copy_(b)
        if i % 3 == 2:
            out = step(state, *fixed)
        else:
            g, out = graphs[i % 2]
            g.replay()
        torch.cuda.synchronize()
        assert same(out[0], want[i][0]) and same(out[1], want[i][1]), i
        step(scratch, *turns[0])
        scratch = fresh()
    assert all(same(a, b) for a, b in zip((*state[0], *state[1], state[2]), end))


def test_threads_that_share_tables():
    """Two threads on one stream and the same tables, calls of two launches: each call is one piece, so no page is dealt twice"""
    P = load("pages")
    S, page, pages, row = 700, 8, 20000, 60
    tables = P.newPageTables(S, row, pages)
    lens, counts = ints([0] * S), [ints([(31 * s + 7 * t) % 400 for s in range(S)]) for t in range(2)]

    def work(t):
        for _ in range(30):
            P.reservePages(tables, lens, 400, page, counts[t])
            P.trimPages(tables, counts[t] // 2, page)
    threads = [threading.Thread(target=work, args=(t,)) for t in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    held, free = tables.held.tolist(), tables.free.tolist()[:tables.freeCount.item()]
    owned = [p for s, line in enumerate(tables.table.tolist()) for p in line[:held[s]]]
    assert sorted(owned + free) == list(range(pages))


def test_calls_of_several_threads_and_streams():
    """Each thread on a stream of its own, long contexts in several parts: the same bits as alone"""
    P, r = load("pages"), maker(11)
    heads, group, dk, page, lens = 2, 4, 128, 64, [20000, 300]
    table = dealt(6, [l + 1 for l in lens], page, 320, 340)
    kv = poisoned(r, table, [l + 1 for l in lens], page, 340, heads, dk, F16)
    q, table, lens = side_by_side(r, 2, heads * group, 1, dk, F16), ints(table), ints(lens)
    want = P.AttentionOverPages(q, kv, table, lens)
    torch.cuda.synchronize()
    wrong = []

    def work(own):
        with torch.cuda.stream(torch.cuda.Stream() if own else torch.cuda.default_stream()):
            for _ in range(20):
                if not same(P.AttentionOverPages(q, kv, table, lens), want):
                    wrong.append(own)
    threads = [threading.Thread(target=work, args=(i % 2 == 0,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong

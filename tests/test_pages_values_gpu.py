"""Attention over pages on the GPU: infinities among the values, wherever the positions that hold them come to lie."""
import pytest
import torch

from conftest import load
from test_pages_gpu import BF16, F16, F32, check, dealt, expected, ints, maker, poisoned, side_by_side

pytestmark = pytest.mark.gpu

INF = float("inf")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dk", [64, 128, 256])
@pytest.mark.parametrize("group,n", [(4, 1), (5, 4), (8, 7), (8, 16)])
@pytest.mark.parametrize("past", [20, 100, 2500])
@pytest.mark.parametrize("low", [200.0, INF])
def test_an_infinity_is_the_result_whatever_its_weight(dtype, dk, group, n, past, low):
    """Queries are ones, so a position's score is the sum of its key, and a key of equal negative numbers makes it as low as wanted: e^-200 of the
    largest weight (2^-288), or nothing.  The low positions are every second 32 (what a wave, or half of the waves, has all of its
    positions among) and the first half of a long sequence (whole parts of it).  A result that sees an infinity there is that infinity, NaN where it sees
    both or NaN, and all other results are as they are without the low positions."""
    pages, r = load("pages"), maker(21)
    heads, page = 2, 16
    row = -(-(past + n) // page)
    table = dealt(8, [past + n], page, row, row)
    kv = poisoned(r, table, [past + n], page, row, heads, dk, dtype)
    at = torch.arange(row * page)
    lows = (at // 32 % 2 == 0) if past < 1000 else at < past // 2
    lows &= at < past - 8
    key = -low / dk ** 0.5
    for j in lows.nonzero()[:, 0].tolist():
        kv.k[table[0][j // page], :, j % page] = key
        kv.v[table[0][j // page], :, j % page] = 0
    q = torch.ones(1, n, heads * group, dk, device="cuda").to(dtype).transpose(1, 2)
    clean = pages.AttentionOverPages(q, kv, ints(table), ints([past]))
    assert torch.isfinite(clean).all()
    first, last = int(lows.nonzero()[0]), int(lows.nonzero()[-1])
    for j, d, x in ((first, 0, INF), (last, 1, -INF), (first, 2, INF), (last, 2, -INF), (last, 3, float("nan")), (last, dk - 1, INF)):
        kv.v[table[0][j // page], 1, j % page, d] = x
    got = pages.AttentionOverPages(q, kv, ints(table), ints([past]))
    assert torch.equal(got[:, :group], clean[:, :group])
    seen = got[0, group:]
    assert (seen[..., 0] == INF).all() and (seen[..., 1] == -INF).all() and torch.isnan(seen[..., 2:4]).all() and (seen[..., dk - 1] == INF).all()
    assert torch.equal(seen[..., 4:dk - 1], clean[0, group:, :, 4:dk - 1])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dk", [64, 128, 256])
@pytest.mark.parametrize("group,n", [(4, 1), (5, 4), (8, 7), (8, 16)])
@pytest.mark.parametrize("past", [20, 100, 2500])
def test_an_infinity_where_all_scores_are_minus_infinity(dtype, dk, group, n, past):
    """Such a token gives zeros, but for the infinities that it sees"""
    pages, r = load("pages"), maker(22)
    heads, page = 2, 16
    row = -(-(past + n) // page)
    table = dealt(9, [past + n], page, row, row)
    kv = poisoned(r, table, [past + n], page, row, heads, dk, dtype)
    kv.k.fill_(-INF)
    q = torch.ones(1, n, heads * group, dk, device="cuda").to(dtype).transpose(1, 2)
    assert not pages.AttentionOverPages(q, kv, ints(table), ints([past])).any()
    for j, d, x in ((3, 0, INF), (past - 1, 1, -INF), (past // 2, 2, float("nan"))):
        kv.v[table[0][j // page], 1, j % page, d] = x
    got = pages.AttentionOverPages(q, kv, ints(table), ints([past]))
    assert not got[:, :group].any() and not got[0, group:, :, 3:].any()
    assert (got[0, group:, :, 0] == INF).all() and (got[0, group:, :, 1] == -INF).all() and torch.isnan(got[0, group:, :, 2]).all()


def test_scores_that_are_no_numbers_beside_infinities():
    """A key of infinities that a query makes NaN of, in another part than the infinity among the values: the whole row is NaN"""
    pages, r = load("pages"), maker(23)
    heads, page, past, dk = 2, 16, 2500, 64
    row = -(-(past + 1) // page)
    table = dealt(10, [past + 1], page, row, row)
    for dtype in (F32, F16, BF16):
        kv = poisoned(r, table, [past + 1], page, row, heads, dk, dtype)
        q = side_by_side(r, 1, heads * 4, 1, dk, dtype)
        kv.v[table[0][0], 1, 5, 9] = INF
        kv.k[table[0][past // page], 1, past % page] = INF
        got = pages.AttentionOverPages(q, kv, ints(table), ints([past]))
        assert torch.isnan(got[0, 4:]).all()
        check(got[:, :4], *expected(q[:, :4], pages.PagedCache(kv.k[:, :1], kv.v[:, :1]), ints(table), [past]))

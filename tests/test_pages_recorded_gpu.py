"""Recorded steps over a cache in pages where they take a workspace and several launches: attention in parts of sequences, pages dealt and taken back
by two launches."""
import pytest
import torch

from conftest import load
from test_pages_gpu import BF16, F16, F32, check, dealt, expected, ints, maker, poisoned, same, side_by_side

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,group,n", [(BF16, 4, 1), (F16, 8, 7), (F32, 4, 6), (F32, 8, 7)])
def test_attention_in_parts_is_replayed(dtype, group, n):
    """Two graphs of attentions over long contexts, replayed at once on two streams beside eager calls, lengths changed in between: a workspace
    each, and every result that of an eager call"""
    pages, r = load("pages"), maker(31)
    S, heads, dk, page = 4, 2, 128, 16
    longest = [3000, 100, 6000, 1]
    row = -(-(6000 + n) // page)
    table = dealt(11, [l + n for l in longest], page, row, 700)
    kv = poisoned(r, table, [l + n for l in longest], page, 700, heads, dk, dtype)
    table = ints(table)
    qs = [side_by_side(r, S, heads * group, n, dk, dtype) for _ in range(2)]
    lens = [ints(longest) for _ in range(2)]
    graphs = []
    for q, l in zip(qs, lens):
        pages.AttentionOverPages(q, kv, table, l)   # (before it is recorded)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = pages.AttentionOverPages(q, kv, table, l)
        graphs.append((g, out))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn, now in enumerate((longest, [2999, 50, 700, 0], [1, 1, 5000, 1], [0, 0, 0, 0], longest)):
        for l in lens:
            l.copy_(ints(now))
        want = [pages.AttentionOverPages(q, kv, table, lens[0]).clone() for q in qs]
        for _, out in graphs:
            out.fill_(9)
        torch.cuda.synchronize()
        for st, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
        eager = pages.AttentionOverPages(qs[0], kv, table, lens[0])
        torch.cuda.synchronize()
        assert same(eager, want[0]), turn
        for (_, out), w in zip(graphs, want):
            assert same(out, w), turn
        check(want[0], *expected(qs[0], kv, table, now))


def test_calls_of_two_launches_are_replayed():
    """Reserving, writing and trimming of many sequences, recorded twice over the same tables, replayed in turn with eager calls between: all as the
    eager ones"""
    P, r = load("pages"), maker(32)
    S, page, n, pages, row, heads, dk = 700, 8, 13, 6000, 9, 1, 16   # (slots past 8192, entries past 4096)
    counts = [ints([(s * 7 + t) % (n + 1) for s in range(S)]) for t in range(2)]
    kept = [(c // 2).to(torch.int32) for c in counts]
    k, v = side_by_side(r, S, heads, n, dk, F16), side_by_side(r, S, heads, n, dk, F16)

    def fresh():
        return P.newPagedCache(pages, heads, page, dk, F16), P.newPageTables(S, row, pages), torch.zeros(S, dtype=torch.int32, device="cuda")

    def step(state, t):
        kv, tables, lens = state
        slots = P.reservePages(tables, lens, n, page, counts[t])
        P.writePages(kv, k, v, slots)
        lens += kept[t]
        lens.masked_fill_(lens > row * page - n, 0)   # (those are done)
        P.trimPages(tables, lens, page)
        return slots
    state, want = fresh(), []
    for turn in range(24):
        slots = step(state, turn % 2)
        want.append([x.clone() for x in (slots, *state[0], *state[1], state[2])])
    scratch, state = fresh(), fresh()
    step(scratch, 0)
    torch.cuda.synchronize()
    graphs = []
    for t in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(state, t)
        graphs.append((g, out))
    for turn in range(24):
        if turn % 5 == 4:
            out = step(state, turn % 2)
        else:
            g, out = graphs[turn % 2]
            g.replay()
        step(scratch, turn % 2)
        torch.cuda.synchronize()
        assert all(same(a, b) for a, b in zip((out, *state[0], *state[1], state[2]), want[turn])), turn

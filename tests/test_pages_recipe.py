"""The decoding step that pages.py's documentation shows, run as it stands there until pages run out and beyond: without a GPU over the
operators as the oracle has them, and on the GPU over the library's.  What the cache holds in front of a sequence's length are always its kept tokens."""
import random as rnd
import textwrap

import pytest
import torch

import pages_oracle as oracle
from conftest import load


def recipe():
    lines = load("pages").__doc__.splitlines()
    first = next(i for i, l in enumerate(lines) if l.startswith("One step of a decoder")) + 1
    last = next(i for i in range(first, len(lines)) if lines[i].strip() and not lines[i].startswith("    "))
    return compile(textwrap.dedent("\n".join(lines[first:last])), "recipe", "exec")


class Layer:
    """what a layer computes around its attention: here given, and passed on"""

    def __init__(self):
        self.qkv, self.seen = None, None

    def project(self, x):
        return self.qkv

    def finish(self, o):
        self.seen = o
        return o


def on_tables(f, tables, *args):
    lists = [t.tolist() for t in tables]
    out = f(*lists, *args)
    for t, x in zip(tables, lists):
        t.copy_(torch.tensor(x, dtype=torch.int32))
    return out


def whole(x):
    return None if x is None else x.tolist()


def oracle_write(cache, k, v, slots):
    page = cache.k.shape[2]
    for s, line in enumerate(slots.tolist()):
        for i, slot in enumerate(line):
            if slot >= 0:
                cache.k[slot // page, :, slot % page], cache.v[slot // page, :, slot % page] = k[s, :, i], v[s, :, i]


ORACLE = {
    "reservePages": lambda tables, lens, n, page, counts=None: torch.tensor(on_tables(oracle.reserve, tables, whole(lens), n, page, whole(counts)),
                                                                             dtype=torch.int32),
    "trimPages": lambda tables, lens, page: on_tables(oracle.trim, tables, whole(lens), page),
    "writePages": oracle_write,
    "AttentionOverPages": lambda q, cache, table, lens, counts=None: oracle.attention(q, *cache, table, whole(lens), whole(counts), q.shape[-1] ** -0.5)[0],
    "rotaryPositions": lambda x, positions, rotary: x,
    "verifyDrafts": lambda tokens, target, numbers, draft=None, parents=None, counts=None: tuple(
        torch.tensor(x, dtype=torch.int32) for x in oracle.verify(tokens.tolist(), target, numbers.tolist(), draft, whole(parents), whole(counts))[:3])}


@pytest.mark.parametrize("n", [5, 1])
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_sequences_that_find_no_pages_stay_where_they_are(device, n):
    pages, kv, rng = load("pages"), load("cache"), rnd.Random(n)
    g = torch.Generator()
    g.manual_seed(n)
    S, heads, group, dk, page, count, row, vocab, L = 4, 2, 2, 16, 8, 7, 6, 9, 2
    ops = ORACLE if device == "cpu" else {**vars(pages), **vars(kv)}
    rows = lambda h: torch.randn(S, n, h, dk, generator=g).to(device).transpose(1, 2)   # noqa: E731
    caches = [pages.newPagedCache(count, heads, page, dk, device=device) for _ in range(L)]
    for c in caches:
        c.k.fill_(float("nan"))
        c.v.fill_(float("nan"))
    tables, layers = pages.newPageTables(S, row, count, device=device), [Layer() for _ in range(L)]
    rotary = None if device == "cpu" else kv.makeRotary(dk)
    lens = torch.zeros(S, dtype=torch.int32, device=device)
    history = [[[] for _ in range(S)] for _ in range(L)]   # keys and values of the kept tokens
    waited = partly = 0
    for turn in range(40):
        for layer in layers:
            layer.qkv = (rows(heads * group), rows(heads), rows(heads))
        numbers, target = torch.rand(S, n, generator=g).to(device), torch.softmax(torch.randn(S, n, vocab, generator=g), -1).to(device)
        tokens = target.argmax(-1).roll(1, 1).to(torch.int32)   # (the target's best ones)
        before = lens.tolist()
        names = {**ops, "torch": torch, "tables": tables, "lens": lens, "n": n, "pageSize": page, "layers": layers, "caches": caches, "rotary": rotary, "x": None,
                 "tokens": tokens, "target": lambda x: target, "random": numbers, "draft": None}
        exec(recipe(), names)
        lens, accepted, following = names["lens"], names["accepted"].tolist(), names["nextTokens"].tolist()
        assert lens.dtype == torch.int32 and lens.tolist() == [b + a for b, a in zip(before, accepted)]
        places = (names["slots"] >= 0).sum(1).tolist()
        table = tables.table.tolist()
        for s in range(S):
            # as many as have a place at the most; one that is settled is kept, and another follows, if one has
            assert (1 <= accepted[s] <= places[s] and 0 <= following[s] < vocab) if places[s] else (accepted[s] == 0 and following[s] == -1)
            waited += places[s] == 0
            partly += 0 < places[s] < n
            for l, (layer, cache, past) in enumerate(zip(layers, caches, history)):
                q, k, v = layer.qkv
                if rotary is not None:
                    k = kv.rotaryPositions(k, torch.tensor(before, dtype=torch.int32, device=device), rotary)
                past[s] += [(k[s, :, i], v[s, :, i]) for i in range(accepted[s])]
                for j, (key, value) in enumerate(past[s]):
                    assert 0 <= table[s][j // page] < count, (turn, s, j)
                    assert torch.equal(cache.k[table[s][j // page], :, j % page], key) and torch.equal(cache.v[table[s][j // page], :, j % page], value)
                assert torch.isfinite(layer.seen[s]).all() and not layer.seen[s, :, places[s]:].any()
        if min(places) == 0 or max(lens.tolist()) > page * row - n:   # one of them is done
            done = rng.randrange(S)
            lens[done] = 0
            for past in history:
                past[done] = []
            ops["trimPages"](tables, lens, page)
    assert waited > 10 and (n == 1 or partly > 0)

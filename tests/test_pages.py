"""A cache in pages and verified drafts, what can be seen without a GPU: the refusals of the C entry points and of the Python operators,
that the parts of an attention stay within grid and workspace, and that the verification's oracle gives the target's distribution."""
import ctypes
import importlib
import math
import os
import random
import subprocess

import pytest
import torch

import pages_oracle as oracle
from conftest import PKG, ROOT, load

GB = 1 << 30
S, H, HQ, N, PAGES, PAGE, ROW, DK, VOCAB = 3, 2, 4, 5, 12, 16, 64, 64, 50000
NAMES = ("k", "v", "table", "held", "free", "count", "lens", "counts", "slots", "xk", "xv", "xq", "qo", "ws", "tokens", "parents", "target", "draft", "random",
         "path", "accepted", "next")
PLACES = {n: (i + 1) * GB for i, n in enumerate(NAMES)}


def dense(heads, n=N, dk=DK):
    return (ctypes.c_int64 * 3)(heads * n * dk, n * dk, dk)


def cache_of(at, **kw):
    g = kw.get
    return load("_lib").Pages(at["k"], at["v"], g("pages", PAGES), g("heads", H), g("page", PAGE), g("dk", DK), g("type", 0))


def tables_of(at, **kw):
    g = kw.get
    return load("_lib").PageTables(at["table"], at["held"], at["free"], at["count"], g("sequences", S), g("row", ROW), g("pages", PAGES))


def reserve(at=PLACES, n=N, page=PAGE, **kw):
    return load("_lib").lib().marian_hip_pages_reserve(ctypes.byref(tables_of(at, **kw)), at["lens"], at["counts"], n, page, at["slots"], None)


def trim(at=PLACES, page=PAGE, **kw):
    return load("_lib").lib().marian_hip_pages_trim(ctypes.byref(tables_of(at, **kw)), at["lens"], page, None)


def write(at=PLACES, n=N, sequences=S, strides=None, **kw):
    st = strides or dense(H)
    return load("_lib").lib().marian_hip_pages_write(ctypes.byref(cache_of(at, **kw)), at["xk"], st, at["xv"], st, sequences, n, at["slots"], None)


def attention(at=PLACES, n=N, sequences=S, row=ROW, q_heads=HQ, scale=0.125, ws_bytes=1 << 40, strides=None, out_strides=None, **kw):
    return load("_lib").lib().marian_hip_pages_attention(
        ctypes.byref(cache_of(at, **kw)), at["table"], sequences, row, at["lens"], at["counts"], n, at["xq"], strides or dense(HQ), q_heads, scale, at["qo"],
        out_strides or dense(HQ), at["ws"], ws_bytes, None)


def verify(at=PLACES, n=N, sequences=S, vocab=VOCAB, type=0, ws_bytes=1 << 40, parents=False, draft=True, strides=None):
    two = ctypes.c_int64 * 2
    x = load("_lib").Drafted(at["tokens"], at["counts"], at["parents"] if parents else None, at["target"], at["draft"] if draft else None, at["random"],
                             sequences, n, vocab, two(*(strides or (n * vocab, vocab))), two((n - 1) * vocab, vocab), type)
    return load("_lib").lib().marian_hip_verify_drafts(ctypes.byref(x), at["path"], at["accepted"], at["next"], at["ws"], ws_bytes, None)


@pytest.mark.parametrize("call,kw,status", [
    (reserve, {"page": 4}, "SHAPE"), (reserve, {"page": 12}, "SHAPE"), (reserve, {"page": 4104}, "SHAPE"), (reserve, {"page": 0}, "SHAPE"),
    (reserve, {"n": -1}, "SHAPE"), (reserve, {"n": 0}, "OK"), (reserve, {"sequences": 0}, "OK"), (reserve, {"sequences": -1}, "SHAPE"),
    (reserve, {"row": 0}, "SHAPE"), (reserve, {"pages": 0}, "SHAPE"), (reserve, {"sequences": 65536}, "RANGE"), (reserve, {"pages": 1 << 26}, "RANGE"),
    (reserve, {"row": 1 << 26}, "RANGE"), (reserve, {"n": (1 << 20) + 1}, "RANGE"), (reserve, {"sequences": 65535, "n": 1 << 20}, "RANGE"),
    (reserve, {"sequences": 65535, "row": 40000}, "RANGE"),
    (trim, {"page": 20}, "SHAPE"), (trim, {"sequences": 0}, "OK"), (trim, {"row": 0}, "SHAPE"), (trim, {"pages": 1 << 26}, "RANGE"),
    (write, {"page": 9}, "SHAPE"), (write, {"type": 3}, "SHAPE"), (write, {"dk": 24}, "SHAPE"), (write, {"dk": 272}, "SHAPE"), (write, {"pages": 0}, "SHAPE"),
    (write, {"heads": 0}, "SHAPE"), (write, {"heads": 4097}, "RANGE"), (write, {"n": -1}, "SHAPE"), (write, {"n": 0}, "OK"), (write, {"sequences": 0}, "OK"),
    (write, {"sequences": 65535, "n": 1 << 20}, "RANGE"), (write, {"strides": (ctypes.c_int64 * 3)(H * N * DK, N * DK, DK + 2)}, "ALIGN"),
    (write, {"strides": (ctypes.c_int64 * 3)(H * N * DK, -DK, DK)}, "SHAPE"),
    (attention, {"page": 7}, "SHAPE"), (attention, {"type": -1}, "SHAPE"), (attention, {"dk": 8}, "SHAPE"), (attention, {"q_heads": 3}, "SHAPE"),
    (attention, {"q_heads": 1}, "SHAPE"), (attention, {"scale": 0.0}, "SHAPE"), (attention, {"scale": math.nan}, "SHAPE"),
    (attention, {"scale": math.inf}, "SHAPE"), (attention, {"row": 0}, "SHAPE"), (attention, {"row": 1 << 26}, "RANGE"), (attention, {"n": -1}, "SHAPE"),
    (attention, {"n": 0}, "OK"), (attention, {"sequences": 0}, "OK"), (attention, {"sequences": 65536}, "RANGE"), (attention, {"ws_bytes": 4096}, "WORKSPACE"),
    (attention, {"n": (1 << 20) + 1}, "RANGE"), (attention, {"sequences": 65535, "heads": 4096, "q_heads": 4096, "n": 1 << 16, "row": 1}, "RANGE"),
    (attention, {"out_strides": (ctypes.c_int64 * 3)(HQ * N * DK, 0, DK)}, "ALIAS"),
    (attention, {"out_strides": (ctypes.c_int64 * 3)(HQ * N * DK, N * DK, DK - 16)}, "ALIAS"),
    (verify, {"n": 0}, "SHAPE"), (verify, {"n": 65}, "SHAPE"), (verify, {"vocab": 0}, "SHAPE"), (verify, {"vocab": 1 << 24}, "RANGE"),
    (verify, {"type": 3}, "SHAPE"), (verify, {"sequences": 65536}, "RANGE"), (verify, {"sequences": 0}, "OK"), (verify, {"parents": True}, "SHAPE"),
    (verify, {"ws_bytes": 100}, "WORKSPACE"), (verify, {"strides": (-1, VOCAB)}, "SHAPE")])
def test_arguments_refused(call, kw, status):
    """(nothing is dereferenced: all is found before any HIP call)"""
    L = load("_lib")
    assert call(**kw) == (L.OK if status == "OK" else getattr(L, "ERR_" + status))


POOL, KV, Q, INTS = 4 * PAGES * H * PAGE * DK, 4 * S * H * N * DK, 4 * S * HQ * N * DK, 4 * S


def sizes(call):
    L = load("_lib").lib()
    ws = L.marian_hip_verify_drafts_workspace_bytes(S, VOCAB) if call is verify else L.marian_hip_pages_attention_workspace_bytes(S, H, HQ, N, DK, 0)
    return {"k": POOL, "v": POOL, "table": INTS * ROW, "held": INTS, "free": 4 * PAGES, "count": 4, "lens": INTS, "counts": INTS, "slots": INTS * N, "xk": KV,
            "xv": KV, "xq": Q, "qo": Q, "ws": ws, "tokens": INTS * N, "parents": INTS * N, "target": 4 * S * N * VOCAB, "draft": 4 * S * (N - 1) * VOCAB,
            "random": INTS * N, "path": INTS * N, "accepted": INTS, "next": INTS}


@pytest.mark.parametrize("call,written,read", [
    (reserve, ["table", "held", "free", "count", "slots"], ["lens", "counts"]), (reserve, ["table"], ["held", "free", "count", "slots"]),
    (reserve, ["held"], ["free", "count", "slots"]), (reserve, ["free"], ["count", "slots"]), (reserve, ["count"], ["slots"]),
    (trim, ["table", "held", "free", "count"], ["lens"]), (trim, ["table"], ["held", "free", "count"]),
    (write, ["k", "v"], ["xk", "xv", "slots"]), (write, ["k"], ["v"]),
    (attention, ["qo", "ws"], ["k", "v", "xq", "table", "lens", "counts"]), (attention, ["qo"], ["ws"]),
    (verify, ["path", "accepted", "next", "ws"], ["tokens", "counts", "target", "draft", "random"]), (verify, ["path"], ["accepted", "next", "ws"]),
    (verify, ["accepted"], ["next", "ws"]), (verify, ["next"], ["ws"])])
def test_overlaps_refused(call, written, read):
    alias, size = load("_lib").ERR_ALIAS, sizes(call)
    for w in written:
        for r in read:
            assert call({**PLACES, w: PLACES[r]}) == alias, (w, r)
            # the end of what is written over the start of what is read
            assert call({**PLACES, w: PLACES[r] - (size[w] - 4) // 256 * 256}) == alias, (w, r)


def test_a_trees_parents_are_not_written_over():
    alias = load("_lib").ERR_ALIAS
    for w in ("path", "accepted", "next", "ws"):
        assert verify({**PLACES, w: PLACES["parents"]}, parents=True, draft=False) == alias


@pytest.mark.parametrize("call,places,may_miss", [
    (reserve, ["table", "held", "free", "count", "lens", "counts", "slots"], ["counts"]), (trim, ["table", "held", "free", "count", "lens"], []),
    (write, ["k", "v", "xk", "xv", "slots"], []), (attention, ["k", "v", "xq", "qo", "table", "lens", "counts", "ws"], ["counts"]),
    (verify, ["tokens", "counts", "target", "draft", "random", "path", "accepted", "next", "ws"], ["counts", "draft"])])
def test_missing_and_misaligned(call, places, may_miss):
    L = load("_lib")
    for p in places:
        if p not in may_miss:
            assert call({**PLACES, p: None}) == L.ERR_NULL, p
        assert call({**PLACES, p: PLACES[p] + 2}) == L.ERR_ALIGN, p


def test_operators_refuse_what_they_do_not_take():
    pages, kv, error = load("pages"), load("cache"), load("_lib").MarianHipError
    cache = pages.newPagedCache(PAGES, H, PAGE, DK, device="cpu")
    tables = pages.newPageTables(S, ROW, PAGES, device="cpu")
    x, lens, slots = torch.zeros(S, H, N, DK), torch.zeros(S, dtype=torch.int32), torch.zeros(S, N, dtype=torch.int32)
    target = torch.full((S, N, 7), 1 / 7)
    calls = [lambda: pages.reservePages(tables, lens, N, PAGE), lambda: pages.trimPages(tables, lens, PAGE),
             lambda: pages.writePages(cache, x, x, slots), lambda: pages.AttentionOverPages(x, cache, tables.table, lens),
             lambda: pages.reservePages(tables[:3], lens, N, PAGE), lambda: pages.writePages(cache[0], x, x, slots),
             lambda: pages.newPagedCache(PAGES, H, PAGE, DK, torch.float64, "cpu"),
             lambda: kv.verifyDrafts(slots, target, torch.zeros(S, N)), lambda: kv.verifyDrafts(slots, target.double(), torch.zeros(S, N)),
             lambda: kv.verifyDrafts(torch.zeros(S, 65, dtype=torch.int32), target, torch.zeros(S, 65)), lambda: kv.verifyDrafts(slots, None, None)]
    for call in calls:
        with pytest.raises(error):
            call()


def test_the_operators_are_exported_under_their_names():
    pages = importlib.import_module(PKG + ".pages")
    for name in ("PagedCache", "PageTables", "newPagedCache", "newPageTables", "reservePages", "trimPages", "writePages", "AttentionOverPages"):
        assert callable(getattr(pages, name))
    assert callable(importlib.import_module(PKG + ".cache").verifyDrafts)


# ---- the plan of the attention ------------------------------------------------------------------------------
PLAN = r"""
#include "pages_plan.h"
#include <cstdio>
int main() {
  long long s, h, hq, n, dk, width;
  while(std::scanf("%lld %lld %lld %lld %lld %lld", &s, &h, &hq, &n, &dk, &width) == 6) {
    const auto p = marian_hip::pages_attention_plan(s, h, hq, n, dk, (int)width);
    std::printf("%d %d %d %d %lld %lld %lld %lld %lld %lld\n", p.dp, p.tile_rows, p.waves, p.least, (long long)p.row_tiles, (long long)p.target,
                (long long)p.items, (long long)p.slots, (long long)p.grid, (long long)marian_hip::pages_attention_bytes(p, h));
  }
}
"""


def test_parts_stay_within_grid_and_workspace(tmp_path):
    """The kernel's division of positions into parts, for lengths of all kinds: never more parts than items, nor more of
    sequences with several than slots, and the workspace holds them; the counters are in its first bytes."""
    (tmp_path / "plan.cpp").write_text(PLAN)
    exe = tmp_path / "plan"
    subprocess.run(["g++", "-std=c++17", "-I", os.path.join(ROOT, PKG, "csrc"), "-o", str(exe), str(tmp_path / "plan.cpp")], check=True)
    rng, cases = random.Random(3), []
    for _ in range(400):
        h = rng.choice([1, 2, 4, 8, 16, 32])
        cases.append((rng.choice([1, 2, 7, 64, 65, 300, 1500, 4100]), h, h * rng.choice([1, 2, 4, 8, 16]), rng.choice([1, 2, 16, 17, 64, 100, 5000]),
                      rng.choice([16, 64, 80, 128, 256]), rng.choice([2, 4])))
    out = subprocess.run([str(exe)], input="\n".join(" ".join(map(str, c)) for c in cases), capture_output=True, text=True, check=True).stdout
    lib = load("_lib").lib()
    for (s, h, hq, n, dk, width), line in zip(cases, out.splitlines()):
        dp, tile, waves, least, tiles, target, items, slots, grid, size = map(int, line.split())
        rows = n * (hq // h)
        assert dp >= dk and tile * tiles >= rows > tile * (tiles - 1) and grid >= items * h * tiles and waves in (1, 4, 8)
        assert lib.marian_hip_pages_attention_workspace_bytes(s, h, hq, n, dk, 0 if width == 4 else 2) == size
        if target == 1:
            assert items == s and slots == 0 and size == 0
            continue
        counters = slots * h * tiles
        assert 4 * counters <= 32768 and size == 32768 + counters * tile * (dp + 1) * 4
        # what the parts are joined through reaches over all of a sequence's, in 32 bits
        assert 64 * h * tiles * (tile * dp + (tile + 3) // 4 * 4) * 4 < 1 << 32
        for longest in (0, 1, 127, 128, 129, 5000, 1 << 20):
            blocks = [(rng.randint(0, longest) + 127) // 128 for _ in range(s)]
            blocks[rng.randrange(s)] = (longest + 127) // 128
            each = max(least, -(-sum(blocks) // target))
            # (up to four blocks stay whole, and 64 parts of a sequence are the most)
            parts = [max(1, -(-b // max(each, 4 if b <= 4 else 0, -(-b // 64)))) for b in blocks]
            several = sum(p for p in parts if p > 1)
            assert sum(parts) <= items and several <= slots and several < 4096, (s, target, longest)


def test_the_shapes_that_are_tested_launch_every_form(tmp_path):
    """What test_pages_gpu.py takes for all forms, against the launcher's choice: type, values of a row, whole or not, sixteens of rows, waves, and
    positions shared in LDS"""
    source = open(os.path.join(ROOT, "tests", "test_pages_gpu.py")).read()
    names = {}
    exec(next(l for l in source.splitlines() if l.startswith("FORMS = ")), names)
    (tmp_path / "plan.cpp").write_text(PLAN.replace('"%d %d %d %d %lld', '"%d %d %d %d %d %d %lld').replace("p.dp, p.tile_rows,", "p.many, p.qt, p.dp, p.tile_rows,"))
    exe = tmp_path / "plan"
    subprocess.run(["g++", "-std=c++17", "-I", os.path.join(ROOT, PKG, "csrc"), "-o", str(exe), str(tmp_path / "plan.cpp")], check=True)
    cases = [(s, 2 if s < 100 else 4, (2 if s < 100 else 4) * group, n, dk, width) for dk, group, n, s in names["FORMS"] for width in (2, 4)]
    out = subprocess.run([str(exe)], input="\n".join(" ".join(map(str, c)) for c in cases), capture_output=True, text=True, check=True).stdout
    got = set()
    for (s, h, hq, n, dk, width), line in zip(cases, out.splitlines()):
        many, qt, dp, tile, waves = map(int, line.split()[:5])
        got.add((width, dp, dk == dp, many, tile // 64 if many else qt, 4 if many else waves))
    want = {(w, dp, whole, 0, qt, waves) for w in (2, 4) for dp in (64, 128, 256) for whole in (True, False) for qt in (1, 2) for waves in (1, 4)
            if not (w == 4 and dp == 256 and qt == 2)}
    want |= {(w, dp, whole, 1, qt, 4) for w, dp in ((2, 64), (2, 128), (4, 128)) for whole in (True, False) for qt in (1, 2)}
    assert got == want


# ---- what the verification gives ----------------------------------------------------------------------------
@pytest.mark.parametrize("form", ["drawn", "best", "tree"])
def test_verified_words_are_distributed_as_the_targets(form):
    """The first two words that come out, over evenly spaced numbers u for every judgement and draw: their frequencies are the target's but for
    the spacing.  (The target's second row depends on the first word, as a model's does.)"""
    words, steps = 3, 24
    first = torch.tensor([0.5, 0.3, 0.2], dtype=torch.float64)
    second = torch.tensor([[0.1, 0.6, 0.3], [0.25, 0.25, 0.5], [0.8, 0.1, 0.1]], dtype=torch.float64)
    thinks = torch.tensor([0.3, 0.2, 0.5], dtype=torch.float64)   # the drafter, in place of `first`
    got = torch.zeros(words, dtype=torch.float64)
    us = (torch.arange(steps, dtype=torch.float64) + 0.5) / steps
    if form == "drawn":
        cases = [([0, w], None, float(thinks[w])) for w in range(words)]
    elif form == "best":
        cases = [([0, 2], None, 1.0)]
    else:
        cases = [([0, 2, 1], [[-1, 0, 0]], 1.0)]
    for tokens, parents, weight in cases:
        n = len(tokens)
        rows = torch.stack([first] + [second[w] for w in tokens[1:]])[None]
        q = thinks[None, None].expand(1, n - 1, words) if form == "drawn" else None
        for u1 in us:
            for u2 in (us if n == 3 else us[:1]):
                for u0 in us:
                    random_ = [[u0, u1, u2][:n]]
                    path, accepted, following, _ = oracle.verify([tokens], rows, random_, q, parents)
                    word = tokens[path[0][1]] if accepted[0] > 1 else following[0]
                    got[word] += weight / (steps * steps * (steps if n == 3 else 1))
    assert torch.allclose(got, first, atol=2.0 / steps)


def test_the_oracles_tables_undo_each_other():
    rng = random.Random(1)
    for _ in range(50):
        s, row, pages, page = rng.randint(1, 9), rng.randint(1, 6), rng.randint(1, 40), 8
        tables = [[[-1] * row for _ in range(s)], [0] * s, list(range(pages)), [pages]]
        lens = [rng.randint(0, 20) for _ in range(s)]
        oracle.reserve(*tables, [0] * s, 20, page, lens)
        before = [[list(r) for r in tables[0]], list(tables[1]), list(tables[2]), list(tables[3])]
        held = [h * page for h in tables[1]]
        slots = oracle.reserve(*tables, held, 11, page)
        owned = [p for r in tables[0] for p in r if p >= 0] + tables[2][:tables[3][0]]
        assert sorted(owned) == list(range(pages)) and len(set(x for r in slots for x in r if x >= 0)) == sum(x >= 0 for r in slots for x in r)
        oracle.trim(*tables, held, page)
        assert tables == before

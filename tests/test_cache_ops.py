"""Keys and values in 8 bits, what can be seen without a GPU: the turns of rotary positions, the refusals of the C entry
points and of the Python operators, and that the parts of an attention stay within the grid and the workspace planned for them."""
import ctypes
import importlib
import math
import os
import random
import subprocess
from fractions import Fraction

import pytest
import torch

import cache_oracle as oracle
from conftest import PKG, ROOT, load

GB = 1 << 30


# ---- rotary turns --------------------------------------------------------------------------------------
@pytest.mark.parametrize("dims,kw", [
    (8, {}), (64, {}), (128, {"base": 500000.0}), (24, {"scaling": "linear", "factor": 4.0}), (128, {"scaling": "base", "factor": 4.0}),
    (64, {"scaling": "bands", "factor": 8.0, "original": 8192}), (128, {"scaling": "bands", "factor": 32.0, "original": 4096, "slow": 2.0, "fast": 16.0})])
def test_turns_are_the_frequencies(dims, kw):
    """A turn is a whole number of 2^-64: off by the 64 bits of the formula above it (1e-15 of the frequency) and half a unit"""
    kv = load("cache")
    r = kv.makeRotary(dims, device="cpu", **kw)
    want, magnitude = oracle.radians(dims, **kw)
    assert r.turns.shape == (dims // 2,) and r.magnitude == pytest.approx(magnitude, rel=1e-15) and r.interleaved is False
    for got, w in zip(r.turns.tolist(), want.tolist()):
        assert abs(Fraction(got, 2 ** 64) - Fraction(w / (2 * math.pi))) <= Fraction(w / (2 * math.pi)) / 10 ** 14 + Fraction(1, 2 ** 65)


def test_turns_of_a_far_position_keep_their_fraction():
    """position * turns mod 2^64 against whole-number arithmetic, at positions where a float32 angle has no fraction left"""
    turns = load("cache").makeRotary(64, device="cpu").turns
    for at in (1, 131071, 2 ** 31 - 1, -5, -2 ** 31):
        got = oracle.angles(turns, torch.tensor(at))
        for g, t in zip(got.tolist(), turns.tolist()):
            f = Fraction(at * t % 2 ** 64, 2 ** 64)
            f = f - 1 if f >= Fraction(1, 2) else f
            assert g == pytest.approx(float(f) * 2 * math.pi, rel=1e-14, abs=1e-18)


@pytest.mark.parametrize("kw", [{"dims": 4}, {"dims": 12}, {"base": 1.0}, {"base": math.inf}, {"scaling": "other"}, {"scaling": "linear", "factor": 0.5},
                                {"scaling": "linear", "factor": math.nan}, {"scaling": "bands", "factor": 2.0},
                                {"scaling": "bands", "factor": 2.0, "original": 10, "slow": 4.0, "fast": 4.0}])
def test_turns_refused(kw):
    with pytest.raises(load("_lib").MarianHipError):
        load("cache").makeRotary(**{"dims": 64, "device": "cpu", **kw})


# ---- refusals --------------------------------------------------------------------------------------------
S, H, HQ, N, CAP, DK = 3, 2, 4, 5, 32, 64
PLACES = {n: (i + 1) * GB for i, n in enumerate(("k", "v", "ks", "vs", "lens", "counts", "parents", "turns", "xk", "xv", "xq", "qo", "ko", "vo",
                                                 "path", "accepted", "new", "ws"))}


def structs(at=PLACES, **kw):
    L = load("_lib")
    g = lambda name, default: kw.get(name, default)
    return (L.KvCache(at["k"], at["v"], at["ks"], at["vs"], g("sequences", S), g("heads", H), g("capacity", CAP), g("dk", DK), g("format", 0)),
            L.Drafts(at["lens"], at["counts"], at["parents"], g("n", N)),
            L.Rotation(at["turns"], g("dims", DK), g("magnitude", 1.0), 0))


def dense(heads, n=N, dk=DK):
    return (ctypes.c_int64 * 3)(heads * n * dk, n * dk, dk)


def append(at=PLACES, type_=0, q=True, rotation=True, q_heads=HQ, strides=None, in_place=False, **kw):
    c, d, r = structs(at, **kw)
    kv, qs = strides or dense(H), dense(HQ)
    return load("_lib").lib().marian_hip_cache_append(
        ctypes.byref(c), ctypes.byref(d), at["xk"], kv, at["xv"], kv, type_, ctypes.byref(r) if rotation else None,
        at["xq"] if q else None, qs, q_heads, (at["xq"] if in_place else at["qo"]) if q else None, qs, None)


def read(at=PLACES, type_=0, **kw):
    c, d, _ = structs(at, **kw)
    return load("_lib").lib().marian_hip_cache_read(ctypes.byref(c), at["lens"], d.n, at["ko"], at["vo"], type_, None)


def attention(at=PLACES, type_=0, q_heads=HQ, scale=0.125, ws_bytes=1 << 40, **kw):
    c, d, _ = structs(at, **kw)
    qs = dense(HQ)
    return load("_lib").lib().marian_hip_cache_attention(ctypes.byref(c), ctypes.byref(d), at["xq"], qs, q_heads, type_, scale, at["qo"], qs,
                                                         at["ws"], ws_bytes, None)


def keep(at=PLACES, path_len=4, **kw):
    c, _, _ = structs(at, **kw)
    return load("_lib").lib().marian_hip_cache_keep(ctypes.byref(c), at["lens"], at["path"], path_len, at["accepted"], at["new"], None)


def rotary(at=PLACES, type_=0, each=0, strides=None, in_place=False, **kw):
    _, d, r = structs(at, **kw)
    g = lambda name, default: kw.get(name, default)
    st = strides or dense(HQ)
    return load("_lib").lib().marian_hip_rotary(at["xq"], st, at["xq"] if in_place else at["qo"], st, type_, g("sequences", S), HQ, d.n, g("dk", DK),
                                                at["lens"], each, ctypes.byref(r), None)


@pytest.mark.parametrize("call", [append, read, attention, keep])
@pytest.mark.parametrize("kw,status", [
    ({"dk": 24}, "SHAPE"), ({"dk": 272}, "SHAPE"), ({"dk": 0}, "SHAPE"), ({"heads": 0}, "SHAPE"), ({"capacity": 0}, "SHAPE"), ({"format": 2}, "SHAPE"),
    ({"sequences": -1}, "SHAPE"), ({"sequences": 65536}, "RANGE"), ({"heads": 4097, "q_heads": 8194}, "RANGE"), ({"capacity": 1 << 25}, "RANGE"),
    ({"sequences": 0}, "OK")])
def test_caches_refused(call, kw, status):
    """(nothing is dereferenced: all is found before any HIP call)"""
    L = load("_lib")
    if call not in (append, attention):
        kw = {k: v for k, v in kw.items() if k != "q_heads"}
    assert call(**kw) == (L.OK if status == "OK" else getattr(L, "ERR_" + status))


@pytest.mark.parametrize("call,kw,status", [
    (append, {"type_": 3}, "SHAPE"), (append, {"n": -1}, "SHAPE"), (append, {"n": 65}, "SHAPE"), (append, {"q_heads": 0}, "SHAPE"),
    (append, {"dims": 72}, "SHAPE"), (append, {"dims": 12}, "SHAPE"), (append, {"dims": 0}, "SHAPE"), (append, {"magnitude": math.nan}, "SHAPE"),
    (append, {"n": 0}, "OK"), (append, {"strides": (ctypes.c_int64 * 3)(H * N * DK, N * DK, DK + 2)}, "ALIGN"),
    (append, {"strides": (ctypes.c_int64 * 3)(H * N * DK, -DK, DK)}, "SHAPE"),
    (read, {"type_": -1}, "SHAPE"), (read, {"n": -1}, "SHAPE"), (read, {"n": 0}, "OK"), (read, {"n": 1 << 30}, "RANGE"),
    (attention, {"type_": 5}, "SHAPE"), (attention, {"q_heads": 3}, "SHAPE"), (attention, {"q_heads": 1}, "SHAPE"), (attention, {"scale": 0.0}, "SHAPE"),
    (attention, {"scale": -1.0}, "SHAPE"), (attention, {"scale": math.inf}, "SHAPE"), (attention, {"scale": math.nan}, "SHAPE"),
    (attention, {"n": 65}, "SHAPE"), (attention, {"n": 0}, "OK"), (attention, {"ws_bytes": 4096}, "WORKSPACE"),
    (keep, {"path_len": -1}, "SHAPE"), (keep, {"path_len": 65}, "SHAPE"),
    (rotary, {"type_": 3}, "SHAPE"), (rotary, {"dk": 20}, "SHAPE"), (rotary, {"dims": 128}, "SHAPE"), (rotary, {"n": 0}, "OK"),
    (rotary, {"sequences": 1 << 16}, "RANGE"), (rotary, {"strides": (ctypes.c_int64 * 3)(HQ * N * DK, N * DK, DK + 1)}, "ALIGN")])
def test_arguments_refused(call, kw, status):
    L = load("_lib")
    assert call(**kw) == (L.OK if status == "OK" else getattr(L, "ERR_" + status))


def needed():
    L = load("_lib").lib()
    return L.marian_hip_cache_attention_workspace_bytes(S, H, HQ, N, DK)


CODES, SCALES, KV, Q, INTS = S * H * CAP * DK, 4 * S * H * CAP, 4 * S * H * N * DK, 4 * S * HQ * N * DK, 4 * S


def sizes():
    return {"k": CODES, "v": CODES, "ks": SCALES, "vs": SCALES, "lens": INTS, "counts": INTS, "parents": INTS * N, "turns": 4 * DK, "xk": KV, "xv": KV,
            "xq": Q, "qo": Q, "ko": KV, "vo": KV, "path": INTS * 4, "accepted": INTS, "new": INTS, "ws": needed()}


cached = ["k", "v", "ks", "vs"]


@pytest.mark.parametrize("call,written,read_", [
    (append, cached, ["lens", "counts", "parents", "turns", "xk", "xv", "xq"]), (append, ["qo"], ["lens", "counts", "parents", "turns", "xk", "xv", "xq"] + cached),
    (read, ["ko", "vo"], cached + ["lens"]), (read, ["ko"], ["vo"]), (attention, ["qo", "ws"], cached + ["xq", "lens", "counts", "parents"]),
    (attention, ["qo"], ["ws"]), (keep, cached + ["new"], ["lens", "path", "accepted"]), (rotary, ["qo"], ["xq", "lens", "turns"])])
def test_overlaps_refused(call, written, read_):
    alias, size = load("_lib").ERR_ALIAS, sizes()
    for w in written:
        for r in read_:
            if not (w == "qo" and r == "xq" and call in (append, rotary)):   # (in place)
                assert call({**PLACES, w: PLACES[r]}) == alias, (w, r)
    for a, b in zip(cached, cached[1:]):
        assert call is rotary or call is attention or call is read or call({**PLACES, a: PLACES[b]}) == alias
    # the end of what is written over the start of what is read
    for w in written:
        for r in read_:
            assert call({**PLACES, w: PLACES[r] - (size[w] - 4) // 256 * 256}) == alias, (w, r)


@pytest.mark.parametrize("call,places", [(append, cached + ["lens", "turns", "xk", "xv", "qo"]), (read, cached + ["lens", "ko", "vo"]),
                                         (attention, cached + ["lens", "xq", "qo", "ws"]), (keep, cached + ["lens", "path", "accepted", "new"]),
                                         (rotary, ["xq", "qo", "lens", "turns"])])
def test_missing_and_misaligned(call, places):
    L = load("_lib")
    for p in places:
        assert call({**PLACES, p: None}) == L.ERR_NULL, p
        assert call({**PLACES, p: PLACES[p] + 2}) == L.ERR_ALIGN, p


def test_operators_refuse_tensors_of_the_cpu():
    kv, error = load("cache"), load("_lib").MarianHipError
    cache = kv.newCache(S, H, CAP, DK, device="cpu")
    x, lens = torch.zeros(S, H, N, DK), torch.zeros(S, dtype=torch.int32)
    r = kv.makeRotary(DK, device="cpu")
    for call in (lambda: kv.rotaryPositions(x, lens, r), lambda: kv.appendToCache(cache, x, x, lens), lambda: kv.readCache(cache, lens, 2),
                 lambda: kv.AttentionOverCache(x, cache, lens), lambda: kv.keepDrafts(cache, lens, torch.zeros(S, 2, dtype=torch.int32), lens)):
        with pytest.raises(error):
            call()
    with pytest.raises(error):
        kv.newCache(S, H, CAP, DK, "int4", device="cpu")


# ---- the plan of the attention ------------------------------------------------------------------------------
PLAN = r"""
#include "cache_plan.h"
#include <cstdio>
int main() {
  long long s, h, hq, cap, n, dk;
  while(std::scanf("%lld %lld %lld %lld %lld %lld", &s, &h, &hq, &cap, &n, &dk) == 6) {
    const auto p = marian_hip::cache_attention_plan(s, h, hq, cap, n, dk);
    std::printf("%d %d %d %lld %lld %lld %lld %lld %lld\n", p.dp, p.tile_rows, p.least, (long long)p.row_tiles, (long long)p.target, (long long)p.items,
                (long long)p.slots, (long long)p.grid, (long long)marian_hip::cache_attention_bytes(p, h));
  }
}
"""


def test_parts_stay_within_grid_and_workspace(tmp_path):
    """The kernel's division of positions into parts, for lengths of all kinds: never more parts than items, nor more of
    sequences with several than slots, and the workspace holds them; the counters are in their first bytes."""
    (tmp_path / "plan.cpp").write_text(PLAN)
    exe = tmp_path / "plan"
    subprocess.run(["g++", "-std=c++17", "-I", os.path.join(ROOT, PKG, "csrc"), "-o", str(exe), str(tmp_path / "plan.cpp")], check=True)
    rng, cases = random.Random(3), []
    for _ in range(400):
        h = rng.choice([1, 2, 4, 8, 16, 32])
        cases.append((rng.choice([1, 2, 7, 64, 65, 300]), h, h * rng.choice([1, 2, 4, 8, 16]), rng.choice([1, 600, 5000, 1 << 20]), rng.choice([1, 2, 16, 17, 64, 100, 5000]),
                      rng.choice([16, 64, 80, 128, 256])))
    out = subprocess.run([str(exe)], input="\n".join(" ".join(map(str, c)) for c in cases), capture_output=True, text=True, check=True).stdout
    lib = load("_lib").lib()
    for (s, h, hq, cap, n, dk), line in zip(cases, out.splitlines()):
        dp, tile, least, tiles, target, items, slots, grid, size = map(int, line.split())
        rows = n * (hq // h)
        assert dp >= dk and tile * tiles >= rows > tile * (tiles - 1) and grid >= items * h * tiles
        assert lib.marian_hip_cache_attention_workspace_bytes(s, h, hq, n, dk) >= size   # (of any capacity)
        if target == 1:
            assert items == s and slots == 0 and size == 0
            continue
        counters = slots * h * tiles
        assert 4 * counters <= 32768 and size == 32768 + counters * tile * (dp + 1) * 4
        for longest in (0, 1, 127, 128, 129, 5000, 1 << 20):
            blocks = [(rng.randint(0, longest) + 127) // 128 for _ in range(s)]
            blocks[rng.randrange(s)] = (longest + 127) // 128
            each = max(least, -(-sum(blocks) // target))
            # (up to four blocks stay whole, and 48 parts of a sequence are the most)
            parts = [max(1, -(-b // max(each, 4 if b <= 4 else 0, -(-b // 48)))) for b in blocks]
            assert sum(parts) <= items and sum(p for p in parts if p > 1) <= slots, (s, target, longest)


def test_the_operators_are_exported_under_their_names():
    kv = importlib.import_module(PKG + ".cache")
    for name in ("KeyValueCache", "Rotary", "newCache", "makeRotary", "rotaryPositions", "appendToCache", "readCache", "AttentionOverCache", "keepDrafts"):
        assert callable(getattr(kv, name))


# ---- rows that are written ------------------------------------------------------------------------------------
@pytest.mark.parametrize("strides,status", [
    ((HQ * N * DK, N * DK, DK), "OK"), ((HQ * N * DK, DK, HQ * DK), "OK"), ((DK, S * DK, S * HQ * DK), "OK"), ((2 * HQ * N * DK, N * DK, DK), "OK"),
    ((0, N * DK, DK), "ALIAS"), ((HQ * N * DK, 0, DK), "ALIAS"), ((HQ * N * DK, N * DK, 0), "ALIAS"), ((HQ * N * DK, N * DK, DK - 16), "ALIAS"),
    ((HQ * N * DK, (N - 1) * DK, DK), "ALIAS"), ((HQ * N * DK - 16, N * DK, DK), "ALIAS")])
def test_rows_that_are_written_share_no_memory(strides, status):
    """(a call that is fine so far is stopped by an argument that is looked at later)"""
    L, st = load("_lib"), (ctypes.c_int64 * 3)(*strides)
    want = getattr(L, "ERR_" + status) if status != "OK" else None
    c, d, r = structs()
    at = PLACES
    far = {**at, "lens": at["lens"] + 2}
    calls = [lambda: L.lib().marian_hip_rotary(at["xq"], dense(HQ), at["qo"], st, 0, S, HQ, N, DK, far["lens"], 0, ctypes.byref(r), None),
             lambda: L.lib().marian_hip_rotary(at["qo"], st, at["qo"], st, 0, S, HQ, N, DK, far["lens"], 0, ctypes.byref(r), None),
             lambda: L.lib().marian_hip_cache_append(ctypes.byref(c), ctypes.byref(d), at["k"], dense(H), at["xv"], dense(H), 0, None, at["xq"], dense(HQ),
                                                     HQ, at["qo"], st, None),
             lambda: L.lib().marian_hip_cache_attention(ctypes.byref(c), ctypes.byref(d), at["xq"], dense(HQ), HQ, 0, 0.125, at["qo"], st, at["ws"] + 2,
                                                        1 << 40, None)]
    for call, later in zip(calls, (L.ERR_ALIGN, L.ERR_ALIGN, L.ERR_ALIAS, L.ERR_ALIGN)):
        assert call() == (later if want is None else want)


def test_launches_past_the_devices_range_are_refused():
    L = load("_lib")
    many = {"sequences": 65535, "heads": 4096, "capacity": 1, "dk": 16}
    assert attention(q_heads=4096, n=1, **many) == L.ERR_RANGE
    assert keep(**many) == L.ERR_RANGE
    assert read(n=1 << 10, **many) == L.ERR_RANGE
    size = L.lib().marian_hip_cache_attention_workspace_bytes
    assert size(1 << 40, 8, 8, 1, 64) == 0 and size(1, 1, 1 << 40, 1, 64) == 0 and size(1, 1, 1, 1 << 62, 64) == 0 and size(1, 8, 8, 1, 64) > 0

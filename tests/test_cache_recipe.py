"""The decoding step that cache.py's documentation shows, run as it stands there: without a GPU over operators that write down
their calls, and on the GPU over two layers against each layer by itself."""
import textwrap

import pytest

from conftest import load


def recipe():
    lines = load("cache").__doc__.splitlines()
    first = next(i for i, l in enumerate(lines) if l.startswith("One step of a decoder with drafted tokens")) + 1
    last = next(i for i in range(first, len(lines)) if lines[i].strip() and not lines[i].startswith("    "))
    return compile(textwrap.dedent("\n".join(lines[first:last])), "recipe", "exec")


class Layer:
    """what a layer computes around its attention: here given, and passed on"""

    def __init__(self, qkv):
        self.qkv, self.seen = qkv, []

    def project(self, x):
        return self.qkv

    def finish(self, o):
        self.seen.append(o)
        return o


def test_every_layer_starts_from_the_same_lengths():
    calls = []
    names = {"appendToCache": lambda cache, k, v, lens, *a, **kw: calls.append(("append", cache, lens)),
             "AttentionOverCache": lambda q, cache, lens, *a, **kw: calls.append(("attention", cache, lens)),
             "keepDrafts": lambda cache, lens, path, accepted: calls.append(("keep", cache, lens)) or lens + accepted,
             "caches": ["a", "b", "c"], "layers": [Layer((0, 0, 0)) for _ in range(3)], "judge": lambda x: (None, 2), "rotary": None, "parents": None,
             "lens": 10, "x": None}
    exec(recipe(), names)
    for what in ("append", "attention", "keep"):
        assert [c[1:] for c in calls if c[0] == what] == [("a", 10), ("b", 10), ("c", 10)]
    assert names["lens"] == 12


@pytest.mark.gpu
def test_two_layers():
    import torch
    kv = load("cache")
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    S, H, G, n, dk, cap = 3, 2, 2, 6, 64, 40
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")   # noqa: E731
    same = lambda a, b: torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))   # noqa: E731
    rows = lambda h: torch.randn(S, n, h, dk, device="cuda", generator=g).transpose(1, 2)   # noqa: E731
    parents, path, accepted = ints([[-1, 0, 0, 1, 3, -1]] * S), ints([[0, 1, 3, 4], [5, 0, 0, 0], [0, 2, 0, 0]]), ints([4, 1, 2])
    layers = [Layer((rows(H * G), rows(H), rows(H))) for _ in range(2)]
    names = {**vars(kv), "caches": [kv.newCache(S, H, cap, dk) for _ in layers], "layers": layers, "judge": lambda x: (path, accepted),
             "rotary": kv.makeRotary(dk), "parents": parents, "lens": ints([0, 7, 20]), "x": None}
    want = [kv.newCache(S, H, cap, dk) for _ in layers]
    lens = names["lens"]
    for _ in range(3):
        exec(recipe(), names)
        for layer, cache in zip(layers, want):
            q, k, v = layer.qkv
            q = kv.appendToCache(cache, k, v, lens, parents, rotary=names["rotary"], q=q)
            assert same(kv.AttentionOverCache(q, cache, lens, parents), layer.seen[-1])
            after = kv.keepDrafts(cache, lens, path, accepted)
        lens = after
        assert torch.equal(names["lens"], lens)
        assert all(same(a, b) for one, other in zip(names["caches"], want) for a, b in zip(one, other))
    assert lens.tolist() == [12, 10, 26]

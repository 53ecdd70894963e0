"""The workspace that an attention over a quantized cache keeps for its stream: given back with the scratch, and made again."""
import pytest
import torch

from conftest import load
from test_cache_forms_gpu import filled, ints, same

pytestmark = pytest.mark.gpu


def step(n, seed):
    kv = load("cache")
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    cache = filled(g, 2, 4, 4000, 128, "int8")
    q = torch.randn(2, n, 16, 128, device="cuda", generator=g).transpose(1, 2)
    lens = ints([4000 - n, 900])
    return lambda: kv.AttentionOverCache(q, cache, lens)


def test_given_back_and_made_again():
    release = load("integer").Backend.releaseScratch
    one, many = step(1, 1), step(200, 2)
    streams = [torch.cuda.Stream() for _ in range(3)]
    want = [one().clone(), many().clone()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):   # (it has a workspace of its own)
        recorded = one()
    torch.cuda.synchronize()
    release()
    before = torch.cuda.memory_allocated()
    for turn in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                for call, w in ((one, want[0]), (many, want[1]), (one, want[0])):
                    got = call()
                    s.synchronize()
                    assert same(got, w)
                    del got
        assert torch.cuda.memory_allocated() > before + (1 << 20)
        release()
        assert torch.cuda.memory_allocated() == before
        recorded.zero_()
        graph.replay()
        assert same(recorded, want[0])

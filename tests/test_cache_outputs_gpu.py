"""Outputs of the operators over a quantized cache lie in memory as their input does: head by head, or the heads of a position side by side."""
import pytest
import torch

from conftest import load
from test_cache_forms_gpu import ints, same

pytestmark = pytest.mark.gpu

S, H, G, n, dk = 3, 2, 2, 5, 64


def side_by_side(x):
    return x.transpose(1, 2).is_contiguous()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_new_tensors_lie_as_the_input(dtype):
    kv = load("cache")
    rotary, lens = kv.makeRotary(dk), ints([0, 3, 9])
    cache = kv.newCache(S, H, 20, dk)
    heads = torch.randn(S, H * G, 2 * n, 2 * dk, device="cuda").to(dtype)             # head by head
    tokens = torch.randn(S, 2 * n, 2 * H * G, dk, device="cuda").to(dtype).transpose(1, 2)   # side by side
    k = torch.randn(S, H, n, dk, device="cuda").to(dtype)
    calls = {"rotary": lambda q: kv.rotaryPositions(q, lens, rotary), "append": lambda q: kv.appendToCache(cache, k, k, lens, rotary=rotary, q=q),
             "attention": lambda q: kv.AttentionOverCache(q, cache, lens)}
    calls["append"](heads[:, :, :n, :dk])
    for name, call in calls.items():
        for q, together in ((heads[:, :, :n, :dk].contiguous(), False), (heads[:, :, :n, dk:], False), (heads[:, :, 1:n + 1, :dk], False),
                            (heads[:, :, ::2, :dk], False), (tokens[:, :H * G, :n].transpose(1, 2).contiguous().transpose(1, 2), True),
                            (tokens[:, :H * G, :n], True), (tokens[:, ::2, n:], True), (off(tokens[:, :H * G, :n]), True), (off(heads[:, :, :n, :dk]), False)):
            out = call(q)
            assert side_by_side(out) == together and out.is_contiguous() != together, (name, q.stride(), out.stride())
            assert same(out, call(q.contiguous()))
        one = call_of_one(kv, name, heads[:, :, 2:3, :dk], cache, k, lens, rotary)
        assert one.is_contiguous() and side_by_side(one)


def off(q):
    """the same next to an address of 16 bytes: copied first"""
    y = torch.zeros(q.numel() + 1, dtype=q.dtype, device=q.device)[1:]
    if side_by_side(q) or q.stride(1) < q.stride(2):
        return y.view(S, n, H * G, dk).transpose(1, 2).copy_(q)
    return y.view(q.shape).copy_(q)


def call_of_one(kv, name, q, cache, k, lens, rotary):
    if name == "append":
        return kv.appendToCache(cache, k[:, :, :1], k[:, :, :1], lens, rotary=rotary, q=q)
    return kv.rotaryPositions(q, lens, rotary) if name == "rotary" else kv.AttentionOverCache(q, cache, lens)

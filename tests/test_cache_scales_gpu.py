"""Attention over a quantized cache whose scales are at the ends of what float32 holds, against 64 bits (cache_forms.py)."""
import pytest
import torch

import cache_forms as forms
import cache_oracle as oracle
from conftest import load
from test_cache_forms_gpu import check, filled, ints, same

pytestmark = pytest.mark.gpu

# one row of an entry and several, in one part and in many, of all numbers of waves and forms
SHAPES = [(2, 2, 1, 1, 64, 500), (1, 1, 1, 1, 128, 9000), (3, 2, 4, 1, 128, 60000), (3, 2, 2, 2, 64, 70000), (2, 1, 12, 1, 256, 3000), (2, 2, 4, 6, 80, 900),
          (2, 1, 1, 60, 64, 700), (1, 2, 2, 64, 128, 5000), (16, 4, 4, 50, 128, 300), (64, 33, 1, 1, 64, 70), (64, 65, 2, 1, 64, 70)]


def batch(S, H, G, n, dk, cap, format, dtype):
    g = torch.Generator(device="cuda")
    g.manual_seed(dk + cap)
    cache = filled(g, S, H, cap, dk, format)
    q = torch.randn(S, n, H * G, dk, device="cuda", generator=g).to(dtype).transpose(1, 2)
    return cache, q, ints([(cap - n, cap // 2, 3)[s % 3] for s in range(S)])


@pytest.mark.parametrize("format", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("S,H,G,n,dk,cap", SHAPES)
def test_values_next_to_the_largest(S, H, G, n, dk, cap, format, dtype):
    """A result lies among its values, however many of them are summed on the way to it"""
    kv = load("cache")
    cache, q, lens = batch(S, H, G, n, dk, cap, format, dtype)
    cache.kScale.mul_(0.01)   # (scores of a few units: all positions count)
    cache.vScale.copy_(1e38 / oracle.TOP[format] * (1 + torch.arange(cap, device="cuda") % 3))
    cache.v.view(torch.uint8)[..., :8] &= 0x7f   # (and their sum grows)
    got = kv.AttentionOverCache(q, cache, lens)
    assert bool(torch.isfinite(got).all())
    check(got, *forms.attention(q, cache, lens))


@pytest.mark.parametrize("format", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("S,H,G,n,dk,cap", SHAPES)
def test_scales_below_zero(S, H, G, n, dk, cap, format, dtype):
    """A value is code * scale whatever the scale's sign, to attention as to reading back"""
    kv = load("cache")
    cache, q, lens = batch(S, H, G, n, dk, cap, format, dtype)
    for flips in (lambda: torch.ones(S, H, cap, device="cuda") * -1, lambda: torch.sign(torch.arange(cap, device="cuda") % 7 - 3.5).expand(S, H, cap)):
        cache.vScale.mul_(flips())
        cache.kScale.mul_(flips())
        check(kv.AttentionOverCache(q, cache, lens), *forms.attention(q, cache, lens))
        k, v = kv.readCache(cache, lens, n)
        at = lens.long()[:, None, None, None] + torch.arange(n, device="cuda")[None, None, :, None]
        for got, codes, scales in ((k, cache.k, cache.kScale), (v, cache.v, cache.vScale)):
            at4 = at.expand(S, H, n, dk)
            assert same(got, codes.float().gather(2, at4) * scales.gather(2, at4[..., 0])[..., None])

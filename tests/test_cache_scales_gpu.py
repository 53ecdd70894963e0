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


@pytest.mark.parametrize("format", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [1e-26, 1e-30, 1e-33, 1e-37])
@pytest.mark.parametrize("S,H,G,n,dk,cap", SHAPES)
def test_values_next_to_the_smallest(S, H, G, n, dk, cap, size, format, dtype):
    """Weights are rounded as those of scales of 1e-30, where all scales are below that: half a step of the smallest float16 at a unit of
    2^9, 16 times at the most above the largest weight, of a code: 2^-25 / 2^9 * 16 = 2^-30 of it.  (The bound has it for the widest scale.)
    float32 itself has steps of 2^-149 at its end, taken once by each of the sums, at most 48 parts and four waves and one position after
    the other, over the power of two that waves are joined by."""
    kv = load("cache")
    cache, q, lens = batch(S, H, G, n, dk, cap, format, dtype)
    cache.vScale.mul_(size)
    want, tol = forms.attention(q, cache, lens)
    far = 2.0 ** -30 * 1e-30 * cap * oracle.TOP[format] + 2.0 ** -149 * 64.0 * 2.0 ** (6 + cap.bit_length())
    check(kv.AttentionOverCache(q, cache, lens), want, tol + far)


@pytest.mark.parametrize("format", ["int8", "e4m3"])
@pytest.mark.parametrize("S,H,G,n,dk,cap", SHAPES)
def test_keys_of_all_sizes(S, H, G, n, dk, cap, format):
    """Keys up to 2^110 by queries as small, and the other way around: scores of a few units"""
    kv = load("cache")
    for k_size, q_size in ((2.0 ** 104, 2.0 ** -105), (2.0 ** -80, 2.0 ** 80)):
        cache, q, lens = batch(S, H, G, n, dk, cap, format, torch.float32)
        cache.kScale.copy_(k_size * 2.0 ** -7 * (1 + torch.arange(cap, device="cuda") % 3))
        q = q * q_size
        check(kv.AttentionOverCache(q, cache, lens), *forms.attention(q, cache, lens))

"""Every form of the attention over a quantized cache on the GPU, for all types of activations and codes, against the same in 64
bits (cache_forms.py; that its cases launch all forms is tested without a GPU, by the plan)."""
import math

import pytest
import torch

import cache_forms as forms
import cache_oracle as oracle
from conftest import load

pytestmark = pytest.mark.gpu

TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def same(a, b):
    return a.shape == b.shape and torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def check(got, want, tol):
    off = ~((got.double() - want).abs() <= tol) & ~(torch.isnan(got) & torch.isnan(want))
    assert not bool(off.any()), "%d of %d off, first at %s: %r, %r +- %r" % (
        off.sum(), off.numel(), off.nonzero()[0].tolist(), got[off][0].item(), want[off][0].item(), tol[off][0].item())


def filled(g, S, H, cap, dk, format):
    """random codes, scales of a factor of e up and down, some of them zero"""
    kv = load("cache")
    cache = kv.newCache(S, H, cap, dk, format)
    for codes, scales in ((cache.k, cache.kScale), (cache.v, cache.vScale)):
        if format == "int8":
            codes.random_(-127, 128, generator=g)
        else:   # (the sign, and a magnitude of up to 0x7e)
            codes.view(torch.uint8).random_(0, 256, generator=g)
            codes.view(torch.uint8)[codes.view(torch.uint8) % 128 == 127] -= 1
        scales.copy_(torch.exp(0.5 * torch.randn(S, H, cap, device="cuda", generator=g)) * 2.0 / oracle.TOP[format])
    cache.vScale[:, :, 2::29] = 0.0
    return cache


def name(c):
    return "%s%d_dp%d_w%d-%dx%d-n%d-dk%d" % (c.form.kind, c.form.rows, c.form.dp, c.form.waves, c.S, c.H, c.n, c.dk)


@pytest.mark.parametrize("format", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("c", forms.CASES, ids=name)
def test_form(c, dtype, format):
    kv = load("cache")
    g = torch.Generator(device="cuda")
    g.manual_seed(c.S + c.n + c.dk)
    cache = filled(g, c.S, c.H, c.cap, c.dk, format)
    lens = ints(forms.lengths(c))
    q = torch.randn(c.S, c.n, c.H * c.G, c.dk, device="cuda", generator=g).to(TYPES[dtype]).transpose(1, 2)
    behind = torch.arange(c.cap, device="cuda")[None] >= lens[:, None] + c.n   # what nobody may see
    for codes, scales in ((cache.k, cache.kScale), (cache.v, cache.vScale)):
        codes.view(torch.uint8).masked_fill_(behind[:, None, :, None], 0x7f)
        scales.masked_fill_(behind[:, None], math.nan)
    # a chain
    got = kv.AttentionOverCache(q, cache, lens)
    check(got, *forms.attention(q, cache, lens))
    assert same(kv.AttentionOverCache(q, cache, lens), got)
    # rows that see a key, or a value, that is not finite, queries that are not, and all others; only some of the tokens are there
    cache.kScale[1, 0, 3] = math.nan
    cache.vScale[c.S - 1, c.H - 1, c.long // 2] = math.nan
    q[2, 0, c.n - 1, c.dk - 1] = math.inf
    q[0, c.G - 1, 0, 0] = math.nan
    counts = ints([(c.n, c.n + 2, c.n, c.n - c.n // 2, 0, 1)[s % 6] for s in range(c.S)])
    for parents in [None] + ([tree(g, c)] if c.tree else []):
        if parents is not None:   # a drafted token that is not finite: in the results of its own branches
            cache.vScale[3 % c.S, 0, lens[3 % c.S] + c.n // 2] = math.nan
        want, tol = forms.attention(q, cache, lens, parents, counts)
        assert bool(torch.isnan(want).any()) and not bool(torch.isnan(want).all())
        got = kv.AttentionOverCache(q, cache, lens, parents, counts)
        check(got, want, tol)
        assert same(kv.AttentionOverCache(q, cache, lens, parents, counts), got)


def tree(g, c):
    """a chain in the first sequence, then trees of a few branches, values that stand for the settled ones among them"""
    i = torch.arange(c.n, device="cuda")
    back = torch.randint(1, 6, (c.S, c.n), device="cuda", generator=g)
    parents = (i - back).clamp_min(-2)
    parents[0] = i - 1
    if c.S > 2:
        parents[2, c.n // 2] = c.n   # (not before its child)
    return parents.to(torch.int32)

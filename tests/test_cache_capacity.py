"""A larger cache around the same sequences: another form of the attention may take them (that the capacities are on both sides of
the rule is asked of the plan without a GPU), with other last bits and the same result within its bound."""
import pytest
import torch

import cache_forms as forms
from conftest import load
from test_cache_forms_gpu import check, filled, ints

SHAPES = [(2, 8, 1, 1, 64, 300), (5, 4, 2, 2, 128, 700), (3, 2, 8, 1, 80, 900), (1, 8, 4, 1, 128, 60)]


def roomy(S, H, cap):
    return max(cap + 1, 400000 // (S * H) + 1)


def test_capacities_on_both_sides(tmp_path):
    said = forms.plans(tmp_path, [(S, H, G, c, n, dk) for S, H, G, n, dk, cap in SHAPES for c in (cap, roomy(S, H, cap))])
    assert [f.kind for f, *_ in said] == ["some", "few"] * len(SHAPES)


@pytest.mark.gpu
@pytest.mark.parametrize("format", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("S,H,G,n,dk,cap", SHAPES)
def test_same_sequences_in_a_larger_cache(S, H, G, n, dk, cap, dtype, format):
    kv = load("cache")
    g = torch.Generator(device="cuda")
    g.manual_seed(cap)
    tight = filled(g, S, H, cap, dk, format)
    wide = kv.newCache(S, H, roomy(S, H, cap), dk, format)
    for small, large in zip(tight, wide):
        large.view(torch.uint8)[:, :, :cap * small.element_size() if small.dim() == 3 else cap] = small.view(torch.uint8)
    q = torch.randn(S, n, H * G, dk, device="cuda", generator=g).to(dtype).transpose(1, 2)
    lens = ints([(cap - n, 0, cap // 2)[s % 3] for s in range(S)])
    want, tol = forms.attention(q, tight, lens)
    for cache in (tight, wide):
        check(kv.AttentionOverCache(q, cache, lens), want, tol)

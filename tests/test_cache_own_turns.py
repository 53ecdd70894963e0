"""Rotary positions by turns that a program makes itself (models whose scaling makeRotary does not know): any whole numbers of 2^-64
of a turn, any finite magnitude."""
import math

import pytest
import torch

import cache_oracle as oracle
from conftest import load


def own(dims, base, factor, original, slow, fast, device):
    """pairs mixed linearly in their index between the two whose turns in `original` positions are fast and slow, as some models are; in 64 bits"""
    pair = lambda turns: dims * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))   # noqa: E731
    low, high = math.floor(pair(fast)), math.ceil(pair(slow))
    turns = []
    for p in range(dims // 2):
        part = min(1.0, max(0.0, (p - low) / (high - low)))
        w = base ** (-2.0 * p / dims)
        turns.append(round(math.ldexp(w * (1 - part + part / factor) / (2 * math.pi), 64)))
    return load("cache").Rotary(torch.tensor(turns, dtype=torch.int64, device=device), 0.1 * math.log(factor) + 1, False)


def test_bands_are_linear_in_the_turns():
    """The formula of makeRotary's bands, and that it is another one than the mixture in the index: by more than a factor of two of a frequency here"""
    kv = load("cache")
    mine, other = kv.makeRotary(64, scaling="bands", factor=8.0, original=8192, device="cpu"), own(64, 10000.0, 8.0, 8192, 1.0, 32.0, "cpu")
    w, magnitude = oracle.radians(64, scaling="bands", factor=8.0, original=8192)
    assert torch.allclose(mine.turns.double() * 2.0 ** -64 * 2 * math.pi, w, rtol=1e-14) and mine.magnitude == pytest.approx(magnitude) == pytest.approx(other.magnitude)
    ratio = mine.turns.double() / other.turns.double()
    assert ratio[0] == pytest.approx(1.0) and ratio[-1] == pytest.approx(1.0) and ratio.min() < 0.5


@pytest.mark.gpu
def test_turned_by_them():
    kv = load("cache")
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    S, H, n, dk, dims = 2, 3, 9, 128, 64
    rotary = own(dims, 10000.0, 8.0, 8192, 1.0, 32.0, "cuda")
    x = torch.randn(S, H, n, dk, device="cuda", generator=g)
    first = [5, 60000]
    got = kv.rotaryPositions(x, torch.tensor(first, dtype=torch.int32, device="cuda"), rotary).cpu().double()
    for s in range(S):
        want = oracle.rotated(x[s].cpu(), torch.arange(n) + first[s], rotary)
        # sine and cosine in float32 with the angle's own rounding (2^-22 together), two products and a sum (2^-23)
        tol = 3 * 2.0 ** -22 * rotary.magnitude * x[s].cpu().double().abs().amax(-1, keepdim=True) * 2 + want.abs() * 2.0 ** -24
        assert ((got[s] - want).abs() <= tol).all()

"""Inputs on which the weights' bits show in the result of an attention over pages, and how far it may be off with the bits that are promised.
Test infrastructure.

Queries are (1, 0, 0, ..) and the scale is 1, so a score is a key's first number: one product, no rounding.  The last token's values are chosen
such that its result is next to zero: three of its positions, of weight one before they are divided by the sum, take away what the others add up to, what is left
of that by the type of the values, and what is left of that.  So its rounding to the type is next to nothing, too, and what is left are the
errors of the other positions' weights."""
import torch

from cache_oracle import HALF

# half a step of what weights enter the product with: bfloat16 and float16 in two terms of 8 and 11 bits (2^-8 and 2^-11 each), float32 in one
WEIGHTS = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -22, torch.bfloat16: 2.0 ** -16}


def inputs(seed, heads, positions, dk, dtype):
    """keys and values [heads, positions, dk] on the CPU; the balancing positions are 0, 1 and 2"""
    g = torch.Generator()
    g.manual_seed(seed)
    k, v = (torch.randn(heads, positions, dk, generator=g).to(dtype) for _ in "kv")
    k[:, :, 0] = (-2 * torch.rand(heads, positions, generator=g)).to(dtype)
    k[:, :3, 0] = 0
    v[:, :3] = 0
    weights = k[:, :, 0].double().exp()
    for j in range(3):
        v[:, j] = -(weights[:, :, None] * v.double()).sum(1).to(dtype)
    return k, v


def result(k, v):
    """[heads, dk] in 64 bits: of a token that sees all positions"""
    p = torch.softmax(k[:, :, 0].double(), -1)
    return (p[:, :, None] * v.double()).sum(1)


def tolerance(k, v):
    """[heads, dk].  A weight's logarithm: score times log2(e) (that factor and the fused product and sum, 2^-23 of it), subtraction of the maximum and the
    carried one's exponent, together 2^-22 of the largest score, and the exponential, 2^-22.  A weight and the weights' sum are off by
    that each, and by half a step of what weights enter with; sums over n positions of products add 2^-23 each, the sums of
    waves and halves and the division 8 more.  float16: what is left of a weight goes down to half a step of 2^-24 at a unit of 2^11; its results to
    half a step of 2^-24."""
    dtype, n = k.dtype, k.shape[1]
    e = k[:, :, 0].double()
    p = torch.softmax(e, -1)
    off = 2 * (e.abs().amax(-1) * 2.0 ** -22 + 2.0 ** -22) + WEIGHTS[dtype] + (n + 8) * 2.0 ** -23
    size = (p[:, :, None] * v.double().abs()).sum(1)
    tol = size * off[:, None] + result(k, v).abs() * HALF[dtype]
    if dtype == torch.float16:
        tol = tol + p.amax(-1)[:, None] * 2.0 ** -36 * v.double().abs().sum(1) + 2.0 ** -25
    return tol


def emulated(k, v, terms):
    """the result with weights that enter the product in so many terms of the type, the first the largest; all else in 64 bits"""
    up = 2.0 ** 11 if k.dtype == torch.float16 else 1.0
    weights = k[:, :, 0].double().exp() * up
    entering, left = torch.zeros_like(weights), weights
    for _ in range(terms):
        term = left.to(k.dtype).double()
        entering, left = entering + term, left - term
    return ((entering[:, :, None] * v.double()).sum(1) / weights.sum(-1, keepdim=True)).to(k.dtype).double()

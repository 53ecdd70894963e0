"""Keys and values in 8 bits, on the HIP library (include/marian_hip_ops.h): rotary positions, a cache that is
quantized as it is written, attention over it for single tokens, chains and trees of drafted ones, and the
accepted drafts' move.

No counterpart in the reference, whose decoder state is float32 (src/models/transformer.h:683-700) and whose
positions are added to the embeddings (:110-117).  Activations are torch tensors on the GPU, float32, float16 or
bfloat16, [sequences, heads, n, dk] as SplitHeads gives them (dk a multiple of 16, up to 256); tensors that are not
laid out in whole rows of 16-byte pieces are copied first.  lens, counts, parents, paths are int32 on the GPU (int64
is converted) and read there: a step needs no synchronisation, and may be recorded into a graph.  New outputs are dense and lie
in memory as their input does: the heads of a position side by side, or head by head.  There is no CPU fallback.

One step of a decoder with drafted tokens:
    for layer, cache in zip(layers, caches):
        q, k, v = layer.project(x)
        q = appendToCache(cache, k, v, lens, parents, rotary=rotary, q=q)
        x = layer.finish(AttentionOverCache(q, cache, lens, parents))
    path, accepted = judge(x)
    for cache in caches:   # (each of them from the lengths that its drafts were written behind)
        newLens = keepDrafts(cache, lens, path, accepted)
    lens = newLens
For one token, or a prompt, parents is None and lens + n the next step's.  The caches of the surviving hypotheses of
a beam are gathered like any decoder state: ops.selectState on the tensors' float32 views.
"""
import ctypes
from typing import NamedTuple

import torch

from . import _lib
from .integer import _abort_if, _host, _on_gpu, _taken

FORMATS = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
ACTIVATIONS = (torch.float32, torch.float16, torch.bfloat16)
SCALINGS = {None: 0, "linear": 1, "base": 2, "bands": 3}
TREE_MAX = 64   # MARIAN_HIP_TREE_MAX


class KeyValueCache(NamedTuple):
    """codes [sequences, heads, capacity, dk] (torch.int8 or torch.float8_e4m3fn) and float32 scales [sequences, heads,
    capacity] of keys and values; a value is code * scale"""
    k: torch.Tensor
    v: torch.Tensor
    kScale: torch.Tensor
    vScale: torch.Tensor


class Rotary(NamedTuple):
    """turns int64 [pairs]: 2^-64 of a turn a position (mod 2^64); the factor of the turned values; whether a pair is
    (2 p, 2 p + 1) or (p, p + pairs)"""
    turns: torch.Tensor
    magnitude: float
    interleaved: bool


def newCache(sequences, heads, capacity, dk, format="int8", device="cuda"):
    """A cache of zeros; format: "int8" or "e4m3"."""
    _abort_if(format not in FORMATS, "newCache: unknown format {}", format)
    shape = (int(sequences), int(heads), int(capacity), int(dk))

    def codes():
        return torch.zeros(shape, dtype=torch.int8, device=device).view(FORMATS[format])
    return KeyValueCache(codes(), codes(), torch.zeros(shape[:3], device=device), torch.zeros(shape[:3], device=device))


def makeRotary(dims, base=10000.0, interleaved=False, scaling=None, factor=1.0, original=None, slow=1.0, fast=32.0, device="cuda"):
    """The turns of `dims` values of a head: pair p by base^(-2 p / dims) radians a position.  scaling, for contexts
    `factor` times as long as the model was made for: "linear" (all slower), "base" (a larger base), "bands" (pairs of
    fewer than `slow` turns in `original` positions slower, of more than `fast` as they are, a mixture linear in the turns in
    between, and a magnitude of 0.1 ln(factor) + 1).  Models that mix otherwise, linearly in the pair's index for one, are a Rotary of their own:
    turns int64 round(frequency / 2 pi * 2^64), a magnitude, and the order of the pairs."""
    _abort_if(scaling not in SCALINGS, "makeRotary: unknown scaling {}", scaling)
    _abort_if(dims < 8 or dims % 8 != 0, "makeRotary: a multiple of 8 values, got {}", dims)
    turns, magnitude = torch.empty(dims // 2, dtype=torch.int64), ctypes.c_double()
    _lib.check(_lib.lib().marian_hip_rotary_turns(turns.data_ptr(), ctypes.addressof(magnitude), dims, base, SCALINGS[scaling], factor,
                                                  original or 0, slow, fast), "makeRotary")
    return Rotary(turns.to(device), magnitude.value, bool(interleaved))


def _rows(x, what, like=None):
    """x in whole rows: [sequences, heads, n, dk] of an activation type, strides of 16-byte pieces"""
    _abort_if(not isinstance(x, torch.Tensor) or x.dtype not in ACTIVATIONS, "{} expects float32, float16 or bfloat16, got {}", what,
              getattr(x, "dtype", type(x)))
    _abort_if(x.dim() != 4, "{} expects [sequences, heads, n, dk], got {}", what, tuple(x.shape))
    _on_gpu(x)
    _abort_if(like is not None and (x.dtype != like.dtype or x.device != like.device), "{}: {} on {} beside {} on {}", what, x.dtype, x.device,
              like.dtype if like is not None else None, like.device if like is not None else None)
    _abort_if(x.shape[3] % 16 != 0 or not 16 <= x.shape[3] <= 256, "{}: rows of a multiple of 16 values up to 256, got {}", what, x.shape[3])
    whole = 16 // x.element_size()
    if x.data_ptr() % 16 == 0 and x.stride(3) == 1 and all(x.stride(i) % whole == 0 for i in range(3) if x.shape[i] > 1):
        return x
    if x.stride(1) < x.stride(2):   # (the heads of a position side by side, as they were)
        return x.transpose(1, 2).clone(memory_format=torch.contiguous_format).transpose(1, 2)
    return x.clone(memory_format=torch.contiguous_format)


def _whole_numbers(t, shape, device, what):
    _abort_if(not isinstance(t, torch.Tensor) or t.dtype not in (torch.int32, torch.int64) or t.device != device, "{}: whole numbers (int32) on {}",
              what, device)
    _abort_if(tuple(t.shape) != tuple(shape), "{}: shape {}, not {}", what, tuple(shape), tuple(t.shape))
    if t.dtype == torch.int64:   # (what 32 bits do not hold stays beyond any length)
        t = t.clamp(-2 ** 31, 2 ** 31 - 1).to(torch.int32)
    return t.contiguous()


def _cache(cache, what):
    _abort_if(not isinstance(cache, tuple) or len(cache) != 4, "{}: a cache is (k, v, kScale, vScale)", what)
    k, v, ks, vs = cache
    _abort_if(k.dtype not in FORMATS.values() or v.dtype != k.dtype or ks.dtype != torch.float32 or vs.dtype != torch.float32,
              "{}: codes are int8 or float8_e4m3fn and scales float32, got {} {} {} {}", what, k.dtype, v.dtype, ks.dtype, vs.dtype)
    _abort_if(k.dim() != 4 or v.shape != k.shape or ks.shape != k.shape[:3] or vs.shape != k.shape[:3],
              "{}: codes [sequences, heads, capacity, dk] and scales [sequences, heads, capacity], got {} {} {} {}", what, tuple(k.shape),
              tuple(v.shape), tuple(ks.shape), tuple(vs.shape))
    _abort_if(not all(t.is_contiguous() for t in cache), "{}: the cache has to be contiguous{}", what, "")
    _on_gpu(k)
    _abort_if(any(t.device != k.device for t in cache), "{}: the cache lies on several devices{}", what, "")
    return KeyValueCache(*cache)


def _drafts(lens, parents, counts, cache, n, what):
    sequences, device = cache.k.shape[0], cache.k.device
    _abort_if(parents is not None and n > TREE_MAX, "{}: a tree of up to {} tokens, got {}", what, TREE_MAX, n)
    return (_whole_numbers(lens, (sequences,), device, what + ": lens"),
            None if parents is None else _whole_numbers(parents, (sequences, n), device, what + ": parents"),
            None if counts is None else _whole_numbers(counts, (sequences,), device, what + ": counts"))


def _rotation(rotary, dk, device, what):
    _abort_if(not isinstance(rotary, tuple) or len(rotary) != 3 or rotary[0].dtype != torch.int64 or rotary[0].dim() != 1 or
              rotary[0].device != device, "{}: rotary is makeRotary(..) on {}", what, device)
    _abort_if(2 * rotary[0].numel() > dk or rotary[0].numel() % 4 != 0, "{}: {} of {} values turned", what, 2 * rotary[0].numel(), dk)
    return Rotary(rotary[0].contiguous(), float(rotary[1]), bool(rotary[2]))


def _out(out, like, what):
    """a tensor to write into: as it is, or refused"""
    _abort_if(out.dtype != like.dtype or out.device != like.device or out.shape != like.shape or _rows(out, what) is not out,
              "{}: the output has to be a {} tensor {} in whole rows", what, like.dtype, tuple(like.shape))
    return out


def rotaryPositions(x, positions, rotary, out=None):
    """x [sequences, heads, n, dk] with the first values of every row turned by its position: positions [sequences] -
    row i of a sequence at positions[s] + i - or [sequences, n]; int64 that 32 bits do not hold are taken as the nearer end.
    out: x itself, or a tensor apart from it; None: a new one that lies in memory as x does."""
    res = _host.rotary(x, positions, rotary, out)
    if res is not None:
        return res
    what = "rotaryPositions"
    x = _rows(x, what)
    each = isinstance(positions, torch.Tensor) and positions.dim() == 2
    at = _whole_numbers(positions, (x.shape[0], x.shape[2]) if each else (x.shape[0],), x.device, what + ": positions")
    rotary = _rotation(rotary, x.shape[3], x.device, what)
    return _taken(_host.rotary(x, at, rotary, None if out is None else _out(out, x, what)), what)


def appendToCache(cache, k, v, lens, parents=None, counts=None, rotary=None, q=None, qOut=None):
    """Quantizes the keys and values of n new tokens a sequence, [sequences, heads, n, dk], into rows lens[s] .. of the
    cache; rotary: keys (and queries q, returned) are turned by their positions on the way, lens[s] + the number of drafted
    tokens a token descends from.  counts [sequences]: only so many of the n are there (the rest of q comes back as
    zeros).  Tokens past the capacity are dropped.  Returns q turned (qOut; None: a new tensor), or None without q."""
    res = _host.cache_append(cache, k, v, lens, parents, counts, rotary, q, qOut)
    if res is not None:
        return None if res is True else res
    what = "appendToCache"
    cache = _cache(cache, what)
    sequences, heads, _, dk = cache.k.shape
    k = _rows(k, what)
    v = _rows(v, what, k)
    n = k.shape[2]
    _abort_if(tuple(k.shape) != (sequences, heads, n, dk) or v.shape != k.shape or k.device != cache.k.device,
              "{}: keys and values {} {} for a cache {}", what, tuple(k.shape), tuple(v.shape), tuple(cache.k.shape))
    lens, parents, counts = _drafts(lens, parents, counts, cache, n, what)
    if rotary is not None:
        rotary = _rotation(rotary, dk, k.device, what)
    _abort_if(q is None and qOut is not None, "{}: an output for queries, and no queries{}", what, "")
    if q is not None:
        q = _rows(q, what, k)
        _abort_if(q.shape[0] != sequences or q.shape[2] != n or q.shape[3] != dk, "{}: queries {} beside keys {}", what, tuple(q.shape),
                  tuple(k.shape))
        if qOut is not None:
            qOut = _out(qOut, q, what)
    res = _taken(_host.cache_append(cache, k, v, lens, parents, counts, rotary, q, qOut), what)
    return None if res is True else res


def readCache(cache, first, n, dtype=torch.float32):
    """Positions first[s] .. first[s] + n - 1 of keys and values, [sequences, heads, n, dk] each, as `dtype`; positions the
    cache does not have are zeros."""
    res = _host.cache_read(cache, first, n, dtype)
    if res is not None:
        return res
    what = "readCache"
    cache = _cache(cache, what)
    _abort_if(dtype not in ACTIVATIONS, "{} gives float32, float16 or bfloat16, not {}", what, dtype)
    _abort_if(n < 0, "{}: {} positions", what, n)
    first = _whole_numbers(first, (cache.k.shape[0],), cache.k.device, what + ": first")
    return _taken(_host.cache_read(cache, first, n, dtype), what)


def AttentionOverCache(q, cache, lens, parents=None, counts=None, scale=None, out=None):
    """softmax(scale * q k) v of n new tokens a sequence over its cache, to which appendToCache has written them: q
    [sequences, q heads, n, dk], q heads a multiple of the cache's (head h reads head h // (q heads / heads)); scale None:
    1 / sqrt(dk).  A token sees the lens[s] settled positions, itself and what it descends from: the tokens before it, or
    with parents [sequences, n] (n <= 64; -1: continues the settled ones) its branch of the tree.  Rows at or past counts[s]
    come out as zeros.  The last bits of a result depend on the batch's lengths and on the cache's sizes, capacity included; a cache with room for
    400000 positions of all heads of all sequences is taken by a form for long contexts (some 2 us more for short ones).  The output lies in
    memory as q does."""
    res = _host.cache_attention(q, cache, lens, parents, counts, scale, out)
    if res is not None:
        return res
    what = "AttentionOverCache"
    cache = _cache(cache, what)
    q = _rows(q, what)
    sequences, heads, _, dk = cache.k.shape
    _abort_if(q.shape[0] != sequences or q.shape[3] != dk or q.shape[1] % heads != 0 or q.device != cache.k.device,
              "{}: queries {} over a cache {}", what, tuple(q.shape), tuple(cache.k.shape))
    lens, parents, counts = _drafts(lens, parents, counts, cache, q.shape[2], what)
    return _taken(_host.cache_attention(q, cache, lens, parents, counts, scale, None if out is None else _out(out, q, what)), what)


def keepDrafts(cache, lens, path, accepted):
    """The accepted drafted tokens become settled: for j < accepted[s], token path[s, j] (path [sequences, up to 64]) moves to
    row lens[s] + j.  Returns the new lens; lens itself stays, for the other layers' caches."""
    res = _host.cache_keep(cache, lens, path, accepted)
    if res is not None:
        return res
    what = "keepDrafts"
    cache = _cache(cache, what)
    sequences, device = cache.k.shape[0], cache.k.device
    _abort_if(not isinstance(path, torch.Tensor) or path.dim() != 2 or path.shape[1] > TREE_MAX, "{}: a path of up to {} tokens a sequence", what,
              TREE_MAX)
    return _taken(_host.cache_keep(cache, _whole_numbers(lens, (sequences,), device, what + ": lens"),
                                   _whole_numbers(path, (sequences, path.shape[1]), device, what + ": path"),
                                   _whole_numbers(accepted, (sequences,), device, what + ": accepted")), what)

"""A cache of keys and values in pages, on the HIP library (include/marian_hip_ops.h): memory that sequences share, dealt out
`pageSize` positions at a time on the GPU, and attention of new tokens over it.

No counterpart in the reference, whose decoder state is one tensor for all sequences (src/models/transformer.h:683-700).  Where
cache.py gives every sequence its capacity, here a sequence has the pages that its length needs, so lengths may differ and
sequences come and go.  Keys and values are of the activations' type, float32, float16 or bfloat16; activations are [sequences, heads, n, dk]
as SplitHeads gives them (dk a multiple of 16, up to 256).  lens, counts are int32 on the GPU (int64 is converted) and read there:
a step needs no synchronisation, and may be recorded into a graph.  There is no CPU fallback.

One step of a decoder, n tokens a sequence (a prompt, one token, or a chain of drafted ones behind the last):
    slots = reservePages(tables, lens, n, pageSize)
    counts = (slots >= 0).sum(1, dtype=torch.int32)     # the tokens that have a place: fewer than n, or none, where the free pages do not reach
    for layer, cache in zip(layers, caches):     # (all layers have the same pages)
        q, k, v = layer.project(x)
        q, k = rotaryPositions(q, lens, rotary), rotaryPositions(k, lens, rotary)
        writePages(cache, k, v, slots)
        x = layer.finish(AttentionOverPages(q, cache, tables.table, lens, counts))
    path, accepted, nextTokens = verifyDrafts(tokens, target(x), random, draft, counts=counts)     # (cache.py; of a prompt, all counts are accepted)
    lens = lens + accepted
    trimPages(tables, lens, pageSize)     # the refused drafts' pages; with lens 0 those of a sequence that is done
Accepted tokens of a chain lie where they are to stay.  Where slots are -1 a sequence found no free pages, and its length must not grow past the
tokens that have a place: with counts as above these are all that is written, seen and verified.  A sequence without any stays where it is
(accepted is 0, its next token -1), and its step is repeated when others are done.

A page belongs to one sequence.  Rows of a table may be copied to read the same pages - hypotheses of a beam that begin alike, say - but
only one of them may be reserved for, written to or trimmed: trimPages would put the pages of each on the stack, and they would be dealt twice.  There is
no move or copy of pages: a beam search whose hypotheses take each other's place has its cache in cache.py, or copies rows itself.  Chains of tokens only: trees
of drafts are for cache.py, too.
"""
from typing import NamedTuple

import torch

from .cache import ACTIVATIONS, _out, _rows, _whole_numbers
from .integer import _abort_if, _host, _on_gpu, _taken


class PagedCache(NamedTuple):
    """keys and values [pages, heads, pageSize, dk]"""
    k: torch.Tensor
    v: torch.Tensor


class PageTables(NamedTuple):
    """int32: the pages of every sequence in order and -1 behind them [sequences, pages in a row], how many they are
    [sequences], a stack of the free ones [pages] and how many these are [1]"""
    table: torch.Tensor
    held: torch.Tensor
    free: torch.Tensor
    freeCount: torch.Tensor


def newPagedCache(pages, heads, pageSize, dk, dtype=torch.float32, device="cuda"):
    """A cache of zeros; pageSize: a multiple of 8."""
    _abort_if(dtype not in ACTIVATIONS, "newPagedCache: float32, float16 or bfloat16, not {}", dtype)
    shape = (int(pages), int(heads), int(pageSize), int(dk))
    return PagedCache(torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device))


def newPageTables(sequences, row, pages, device="cuda"):
    """Tables of `sequences` sequences of up to `row` pages; all `pages` pages are free, the first ones go first."""
    return PageTables(torch.full((int(sequences), int(row)), -1, dtype=torch.int32, device=device),
                      torch.zeros(int(sequences), dtype=torch.int32, device=device),
                      torch.arange(int(pages) - 1, -1, -1, dtype=torch.int32, device=device),
                      torch.full((1,), int(pages), dtype=torch.int32, device=device))


def _tables(tables, what):
    _abort_if(not isinstance(tables, tuple) or len(tables) != 4 or any(not isinstance(t, torch.Tensor) or t.dtype != torch.int32 for t in tables),
              "{}: tables are (table, held, free, freeCount), int32", what)
    table, held, free, count = tables
    _abort_if(table.dim() != 2 or held.shape != table.shape[:1] or free.dim() != 1 or tuple(count.shape) != (1,) or
              not all(t.is_contiguous() for t in tables), "{}: dense tensors [sequences, row], [sequences], [pages] and [1], got {} {} {} {}", what,
              tuple(table.shape), tuple(held.shape), tuple(free.shape), tuple(count.shape))
    _on_gpu(table)
    _abort_if(any(t.device != table.device for t in tables), "{}: the tables lie on several devices{}", what, "")
    return PageTables(*tables)


def _pages(cache, what):
    _abort_if(not isinstance(cache, tuple) or len(cache) != 2 or any(not isinstance(t, torch.Tensor) for t in cache), "{}: a cache is (k, v)", what)
    k, v = cache
    _abort_if(k.dtype not in ACTIVATIONS or v.dtype != k.dtype, "{}: a cache of float32, float16 or bfloat16, got {} {}", what, k.dtype, v.dtype)
    _abort_if(k.dim() != 4 or v.shape != k.shape or not (k.is_contiguous() and v.is_contiguous()),
              "{}: keys and values are dense [pages, heads, pageSize, dk], got {} {}", what, tuple(k.shape), tuple(v.shape))
    _on_gpu(k)
    _abort_if(v.device != k.device, "{}: the cache lies on several devices{}", what, "")
    return PagedCache(k, v)


def reservePages(tables, lens, n, pageSize, counts=None):
    """Deals pages to the sequences for n new tokens each (counts [sequences]: only so many of them) behind their lens, in the sequences'
    order, and returns where the tokens lie, int32 [sequences, n]: page * pageSize + place; -1 for tokens that are not there, and for all that
    need a new page in a sequence that there are none for (or whose row is too short): pages are dealt to a sequence whole or not at
    all, and once they do not reach for one, to none behind it.  The tables are changed in place."""
    slots = _host.pages_reserve(tables, lens, n, pageSize, counts)
    if slots is not None:
        return slots
    what = "reservePages"
    tables = _tables(tables, what)
    sequences, device = tables.held.shape[0], tables.table.device
    _abort_if(n < 0, "{}: {} tokens", what, n)
    lens = _whole_numbers(lens, (sequences,), device, what + ": lens")
    counts = None if counts is None else _whole_numbers(counts, (sequences,), device, what + ": counts")
    return _taken(_host.pages_reserve(tables, lens, n, pageSize, counts), what)


def trimPages(tables, lens, pageSize):
    """Takes back the pages that lie behind the sequences' lens (0: all of a sequence's).  With the lens of a reservePages it undoes that, if no
    sequence held pages behind its lens before.  No page may be in two sequences' rows (their held pages): it would be dealt twice."""
    if _host.pages_trim(tables, lens, pageSize) is None:
        what = "trimPages"
        tables = _tables(tables, what)
        lens = _whole_numbers(lens, (tables.held.shape[0],), tables.table.device, what + ": lens")
        _taken(_host.pages_trim(tables, lens, pageSize), what)


def writePages(cache, k, v, slots):
    """Writes keys and values [sequences, heads, n, dk] of the cache's type to the slots [sequences, n] that reservePages gave; those below
    0 or past the cache are dropped.  No two tokens have the same slot."""
    if _host.pages_write(cache, k, v, slots) is None:
        what = "writePages"
        cache = _pages(cache, what)
        k = _rows(k, what, cache.k)
        v = _rows(v, what, cache.k)
        _abort_if(v.shape != k.shape or k.shape[1] != cache.k.shape[1] or k.shape[3] != cache.k.shape[3], "{}: keys and values {} {} for a cache {}", what,
                  tuple(k.shape), tuple(v.shape), tuple(cache.k.shape))
        slots = _whole_numbers(slots, (k.shape[0], k.shape[2]), k.device, what + ": slots")
        _taken(_host.pages_write(cache, k, v, slots), what)


def AttentionOverPages(q, cache, table, lens, counts=None, scale=None, out=None):
    """softmax(scale * q k) v of n new tokens a sequence over the pages that writePages has written them to: q [sequences, q heads, n, dk] of
    the cache's type, q heads a multiple of the cache's (head h reads head h // (q heads / heads)); table int32 [sequences, pages in a
    row]; scale None: 1 / sqrt(dk).  A token sees the lens[s] positions before the new ones, itself and the new tokens before it.  Rows of
    the table may share pages; positions of pages that are none (-1), or past the row, are not seen, and a token that sees nothing gives zeros, as do
    rows at or past counts[s].  The last bits of a result depend on the batch's lengths and the table's width.  Made for few rows a head of keys
    (n times the heads that share it): 128 of them read the pages once, or 32 (float32 with dk up to
    64, 16-bit types with dk past 128), or 16 (float32 with dk past 128).  A long sequence among more than 1024, or beside a prompt in the
    same call, is not split over the card: it is better given a call of its own.  An infinity among the values that a token sees is its result,
    whatever its weight.  The output lies in memory as q does."""
    res = _host.pages_attention(q, cache, table, lens, counts, scale, out)
    if res is not None:
        return res
    what = "AttentionOverPages"
    cache = _pages(cache, what)
    q = _rows(q, what, cache.k)
    sequences, heads = q.shape[0], cache.k.shape[1]
    _abort_if(q.shape[3] != cache.k.shape[3] or heads == 0 or q.shape[1] % heads != 0, "{}: queries {} over a cache {}", what, tuple(q.shape),
              tuple(cache.k.shape))
    _abort_if(not isinstance(table, torch.Tensor) or table.dim() != 2, "{}: a table [sequences, pages in a row]{}", what, "")
    table = _whole_numbers(table, (sequences, table.shape[1]), q.device, what + ": table")
    lens = _whole_numbers(lens, (sequences,), q.device, what + ": lens")
    counts = None if counts is None else _whole_numbers(counts, (sequences,), q.device, what + ": counts")
    return _taken(_host.pages_attention(q, cache, table, lens, counts, scale, None if out is None else _out(out, q, what)), what)

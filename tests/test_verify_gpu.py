"""Verification of drafted tokens on the GPU, against the same written out in 64 bits on the CPU (pages_oracle.py)."""
import random

import pytest
import torch

import pages_oracle as oracle
from conftest import load

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def inputs(seed, S, n, vocab, dtype, form, sharp=2.0):
    """probabilities, tokens that are kept about every other time, numbers"""
    g = torch.Generator()
    g.manual_seed(seed)
    logits = sharp * torch.randn(S, n, vocab, generator=g)
    target = torch.softmax(logits, -1).to(dtype)
    near = logits[:, :n - 1] + 0.5 * torch.randn(S, n - 1, vocab, generator=g)
    draft = torch.softmax(near, -1)
    tokens = torch.randint(0, vocab, (S, n), generator=g)
    parents = None
    if form == "drawn":
        if n > 1:
            tokens[:, 1:] = torch.multinomial(draft.view(-1, vocab), 1, generator=g).view(S, n - 1)
    elif form == "best":
        tokens[:, 1:] = near.argmax(-1)
    else:
        rng = random.Random(seed)
        parents = torch.full((S, n), -1, dtype=torch.int32)
        for s in range(S):
            for i in range(1, n):
                p = rng.randint(max(0, i - 4), i - 1)
                parents[s, i] = p
                tokens[s, i] = near[s, p].topk(min(3, vocab)).indices[rng.randrange(min(3, vocab))]   # (siblings may be the same word)
    return tokens.to(torch.int32), target, torch.rand(S, n, generator=g), draft.to(dtype) if form == "drawn" else None, parents


def check(tokens, target, numbers, draft=None, parents=None, counts=None, on_gpu=None):
    kv = load("cache")
    path, accepted, following, near = oracle.verify(tokens.tolist(), target, numbers.tolist(), draft, None if parents is None else parents.tolist(), counts)
    # (sums of up to 2^20 numbers in another order differ by 2^-33 of themselves: what lies nearer to a border could fall on either side)
    assert near > 2.0 ** -33
    up = lambda x: None if x is None else x.cuda()
    got = kv.verifyDrafts(up(tokens), up(target) if on_gpu is None else on_gpu, up(numbers), up(draft), up(parents), None if counts is None else ints(counts))
    assert [x.dtype for x in got] == [torch.int32] * 3
    assert got[0].tolist() == path and got[1].tolist() == accepted and got[2].tolist() == following
    return accepted


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("form", ["drawn", "best", "tree"])
@pytest.mark.parametrize("S,n,vocab", [(1, 1, 1), (1, 1, 7), (5, 2, 2), (7, 4, 33), (3, 64, 100), (9, 6, 1000), (4, 5, 4095), (4, 5, 4096), (4, 5, 4097),
                                       (4, 5, 1023), (4, 5, 1024), (4, 5, 1025), (3, 5, 8191), (3, 5, 8192), (3, 5, 8193), (2, 4, 32767), (2, 4, 32768), (2, 4, 32769), (1, 4, 65537),
                                       (2, 3, 50001), (1, 5, 131071)])
def test_verified(dtype, form, S, n, vocab):
    x = inputs(S + n + vocab, S, n, vocab, dtype, form)
    kept = check(*x)
    assert form != "drawn" or S * n < 20 or max(kept) > 1   # (some are kept; the drafter's best have few of the target's words)
    counts = [(3 * s) % (n + 2) - (s % 2) for s in range(S)]
    check(*x, counts=counts)
    # rows of a wider tensor that start anywhere, and the same row for all
    wide = torch.full((S, n, vocab + 5), 9.0, dtype=dtype, device="cuda")
    wide[..., 3:vocab + 3] = x[1].cuda()
    check(*x, on_gpu=wide[..., 3:vocab + 3])
    check(x[0], x[1][:, :1].expand(S, n, vocab), x[2], None, x[4], on_gpu=x[1].cuda()[:, :1].expand(S, n, vocab))


def test_more_sequences_than_counters():
    torch.manual_seed(3)
    check(*inputs(1, 9000, 2, 4100, BF16, "best"))
    _, target, _, _, _ = inputs(2, 1, 2, 33000, F16, "best")
    tokens, numbers = torch.randint(0, 33000, (9000, 2), dtype=torch.int32), torch.rand(9000, 2)
    tokens[:, 1] = target[0, 0].argmax()
    check(tokens, target.expand(9000, 2, 33000), numbers, on_gpu=target.cuda().expand(9000, 2, 33000))


def test_certain_and_impossible_tokens():
    kv = load("cache")
    S, n, vocab = 6, 4, 300
    tokens, target, numbers, draft, _ = inputs(3, S, n, vocab, F32, "drawn")
    sure = torch.zeros(S, n, vocab)
    sure[:, torch.arange(n - 1), 7], sure[:, n - 1, 11] = 1.0, 1.0
    tokens[:, 1:] = 7
    path, accepted, following = kv.verifyDrafts(tokens.cuda(), sure.cuda(), numbers.cuda(), sure[:, :n - 1].cuda())
    assert accepted.tolist() == [n] * S and following.tolist() == [11] * S and path.tolist() == [[0, 1, 2, 3]] * S
    # a word that is not one, that the target does not have, that nobody has; numbers 0; a residual of nothing (p = q): drawn from p
    for token, q in ((-5, draft), (vocab, draft), (2 ** 31 - 1, None), (8, None), (8, sure[:, :n - 1])):
        tokens[:, 1] = token
        numbers[:, 1:] = 0.0
        path, accepted, following = kv.verifyDrafts(tokens.cuda(), sure.cuda(), numbers.cuda(), None if q is None else q.cuda())
        assert accepted.tolist() == [1] * S and following.tolist() == [7] * S
    # drawing with 0: the first word that has anything; next to 1: the last
    flat = torch.zeros(2, 1, 9000)
    flat[:, 0, [5, 4500, 8998]] = torch.tensor([0.25, 0.5, 0.25])
    got = kv.verifyDrafts(ints([[0], [0]]), flat.cuda(), torch.tensor([[0.0], [1 - 2.0 ** -24]]).cuda())
    assert got[2].tolist() == [5, 8998]
    # borders themselves: 0.25 and 0.75 belong to the next word
    got = kv.verifyDrafts(ints([[0], [0]]), flat.cuda(), torch.tensor([[0.25], [0.75]]).cuda())
    assert got[2].tolist() == [4500, 8998]


def test_what_is_no_probability_counts_as_none():
    kv = load("cache")
    for vocab in (100, 9000, 40000):
        target = torch.zeros(4, 2, vocab)
        target[0, 0, 3] = float("nan")
        target[0, 0, 4] = 0.5
        target[1, 0, 5], target[1, 0, vocab - 2] = -2.0, 1e-30
        target[3] = float("nan")
        got = kv.verifyDrafts(ints([[0, 3], [0, 5], [0, 1], [0, 1]]), target.cuda(), torch.full((4, 2), 0.3).cuda())
        assert got[1].tolist() == [1] * 4 and got[2].tolist() == [4, vocab - 2, -1, -1]
        target[3, 0, 8] = float("inf")
        got = kv.verifyDrafts(ints([[0, 3]] * 4), target.cuda(), torch.full((4, 2), 0.3).cuda())
        assert 0 <= got[2][3].item() < vocab


@pytest.mark.parametrize("vocab", [40, 5000, 40000])
def test_a_draft_that_is_no_distribution(vocab):
    """Nothing left of the target behind a refused draft, over one share of words and many; draft's numbers below zero and NaN"""
    tokens, target, _, draft, _ = inputs(11, 5, 3, vocab, F32, "drawn")
    big = draft * 0 + 2.0
    numbers = torch.tensor([[u, 0.9, 0.9] for u in (0.0, 0.2, 0.5, 0.9, 1 - 2.0 ** -24)])
    check(tokens, target, numbers, big)
    big[:, :, ::3] = float("nan")
    big[:, :, 1::3] = -1.0
    check(tokens, target, numbers, big)


def test_trees_whose_parents_are_odd():
    """Tokens whose parent is none, themselves or behind them are never reached; the first token's own parent says nothing"""
    tokens, target, numbers, _, _ = inputs(4, 1, 6, 50, F32, "best")
    for parents in ([[3, 1, 9, -7, 0, 4]], [[-1, -1, -1, -1, -1, -1]], [[-1, 0, 0, 0, 0, 0]], [[0, 0, 1, 2, 3, 4]], [[5, 2, 0, 2, 3, 4]]):
        check(tokens, target, torch.zeros(1, 6) + 1e-6, None, torch.tensor(parents, dtype=torch.int32))
        check(tokens, target, numbers, None, torch.tensor(parents, dtype=torch.int32))


def test_words_are_distributed_as_the_targets():
    """60000 sequences of one drawn and one best draft: counts of the words that come out are within 5 standard deviations"""
    kv = load("cache")
    S, g = 60000, torch.Generator(device="cuda")
    g.manual_seed(5)
    p = torch.tensor([0.4, 0.05, 0.25, 0.2, 0.1], device="cuda")
    q = torch.tensor([0.1, 0.3, 0.3, 0.2, 0.1], device="cuda")
    target, draft = p.expand(S, 2, 5), q.expand(S, 1, 5)
    for drawn in (True, False):
        tokens = torch.zeros(S, 2, dtype=torch.int32, device="cuda")
        tokens[:, 1] = torch.multinomial(q.expand(S, 5), 1, generator=g)[:, 0].int() if drawn else 1
        path, accepted, following = kv.verifyDrafts(tokens, target, torch.rand(S, 2, device="cuda", generator=g), draft if drawn else None)
        first = torch.where(accepted > 1, tokens[:, 1], following)
        got = torch.bincount(first.long(), minlength=5).double()
        assert ((got - S * p).abs() < 5 * (S * p * (1 - p)).sqrt()).all()


def test_refusals():
    kv, error = load("cache"), load("_lib").MarianHipError
    tokens, target, numbers, draft, parents = [None if x is None else x.cuda() for x in inputs(6, 2, 3, 50, F32, "drawn")]
    tree = ints([[-1, 0, 0]] * 2)
    for call in (lambda: kv.verifyDrafts(tokens, target, numbers, draft, tree), lambda: kv.verifyDrafts(tokens, target[:, :2], numbers),
                 lambda: kv.verifyDrafts(tokens, target, numbers, draft[:, :1]), lambda: kv.verifyDrafts(tokens, target, numbers, draft.half()),
                 lambda: kv.verifyDrafts(tokens, target, numbers.double()), lambda: kv.verifyDrafts(tokens, target, numbers[:, :2]),
                 lambda: kv.verifyDrafts(tokens.float(), target, numbers), lambda: kv.verifyDrafts(tokens, target, numbers, counts=ints([1])),
                 lambda: kv.verifyDrafts(tokens, target, numbers, parents=tree[:, :2]), lambda: kv.verifyDrafts(tokens.cpu(), target, numbers)):
        with pytest.raises(error):
            call()
    want = kv.verifyDrafts(tokens, target, numbers, draft)
    got = kv.verifyDrafts(tokens.long(), target.transpose(0, 1).contiguous().transpose(0, 1), numbers, draft.transpose(1, 2).contiguous().transpose(1, 2))
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    assert [x.shape[0] for x in kv.verifyDrafts(tokens[:0], target[:0], numbers[:0])] == [0, 0, 0]


@pytest.mark.parametrize("vocab", [20000, 70000])
def test_recorded_and_beside_each_other(vocab):
    """Two graphs on streams of their own, replayed together with eager calls between: a workspace each"""
    kv = load("cache")
    first, second = ([None if x is None else x.cuda() for x in inputs(s, 8, 5, vocab, F32, "drawn")] for s in (7, 8))
    want = [[t.clone() for t in kv.verifyDrafts(*x)] for x in (first, second)]
    graphs = []
    for x in (first, second):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = kv.verifyDrafts(*x)
        graphs.append((g, out))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(5):
        for _, out in graphs:
            for t in out:
                t.fill_(-9)
        torch.cuda.synchronize()
        for st, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
        eager = kv.verifyDrafts(*first)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, want[0])), turn
        for (_, out), w in zip(graphs, want):
            assert all(torch.equal(a, b) for a, b in zip(out, w)), turn


def test_a_step_with_drafts_over_a_quantized_cache():
    """append, attention, verification and the accepted drafts' move, as the documentation of the cache has them: what stays in the cache are the
    kept tokens in their order"""
    kv = load("cache")
    S, heads, dk, n, cap, vocab = 3, 2, 64, 7, 64, 400
    g = torch.Generator(device="cuda")
    g.manual_seed(9)
    cache = kv.newCache(S, heads, cap, dk, "int8")
    lens = ints([0, 0, 0])
    history = [[] for _ in range(S)]
    for turn in range(4):
        tokens, target, numbers, _, parents = [None if x is None else x.cuda() for x in inputs(20 + turn, S, n, vocab, F32, "tree", sharp=6.0)]
        k, v, q = (torch.randn(S, heads, n, dk, device="cuda", generator=g) for _ in "kvq")
        kv.appendToCache(cache, k, v, lens, parents)
        assert torch.isfinite(kv.AttentionOverCache(q, cache, lens, parents)).all()
        path, accepted, following = kv.verifyDrafts(tokens, target, numbers, parents=parents)
        lens = kv.keepDrafts(cache, lens, path, accepted)
        for s in range(S):
            history[s] += [k[s, :, i] for i in path[s].tolist() if i >= 0]
        assert lens.tolist() == [len(h) for h in history] and (following >= 0).all()
    assert max(len(h) for h in history) > 4
    for s in range(S):
        got = kv.readCache(cache, ints([0] * S), len(history[s]))[0][s]
        want = torch.stack(history[s], 1)
        assert ((got - want).abs() <= want.abs().amax(-1, keepdim=True) / 127 * 0.51).all()

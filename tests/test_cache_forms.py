"""That the shapes of cache_forms.py launch every form of the attention over a quantized cache, by its plan, and that its attention in
64 bits is cache_oracle's (without a GPU)."""
import pytest
import torch

import cache_forms as forms
import cache_oracle as oracle


def test_every_form_is_launched_by_a_case(tmp_path):
    """(a rule of the plan that moves a case to another form fails here, before its GPU test says nothing about the form any more)"""
    said = forms.plans(tmp_path, [(c.S, c.H, c.G, c.cap, c.n, c.dk) for c in forms.CASES])
    assert len(said) == len(forms.CASES)
    for c, (form, least, target, tiles) in zip(forms.CASES, said):
        assert form == c.form, (c, form)
        assert max(forms.lengths(c)) == c.long and 0 < c.long <= c.cap - c.n
        assert not c.split or max(forms.parts(least, target, forms.lengths(c), c.n, c.cap)) > 1, c
    assert {c.form for c in forms.CASES} == set(forms.FORMS)
    # of both kinds of masks, whole and partly filled tiles of rows
    for f in forms.FORMS:
        mine = [c for c in forms.CASES if c.form == f]
        assert any(c.tree for c in mine) or f.kind == "few" and f.rows == 1
        assert f.kind != "many" or any(c.n * c.G % (64 * f.rows) for c in mine)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("S,H,G,n,dk,cap,tree,counted", [
    (3, 2, 1, 1, 16, 40, False, False), (4, 1, 3, 5, 32, 300, True, False), (3, 2, 2, 6, 16, 20, True, True), (2, 1, 1, 9, 48, 30, False, True)])
def test_the_batched_attention_is_the_oracles(dtype, S, H, G, n, dk, cap, tree, counted):
    """one formula written twice: apart by the order of 64-bit sums, bounds by sums of the positive"""
    g = torch.Generator().manual_seed(S + n)
    cache = [torch.randint(-127, 128, (S, H, cap, dk), generator=g).to(torch.int8) for _ in "kv"] + [
        0.01 * (1 + torch.rand(S, H, cap, generator=g)) for _ in "kv"]
    q = torch.randn(S, H * G, n, dk, generator=g).to(dtype)
    lens = torch.tensor([(0, cap - n, 7, cap - 2)[s % 4] for s in range(S)])
    parents = torch.randint(-2, n + 2, (S, n), generator=g) if tree else None
    counts = torch.tensor([(n, 0, n - 1, 1)[s % 4] for s in range(S)]) if counted else None
    want, far = oracle.attention(q, cache[0].double(), cache[1].double(), cache[2], cache[3], lens, parents, counts, dk ** -0.5)
    got, mine = forms.attention(q, cache, lens, parents, counts, rounding=2.0 ** -22 if dtype == torch.float32 else 2.0 ** -11)
    assert (got - want).abs().max() < 1e-12
    there = (far > 0).any(-1, keepdim=True).expand_as(far)   # (rows that are not there are zeros, and so is their bound)
    if dtype == torch.float16:   # (here with its smallest step, which the oracle's results do not come down to)
        far = far + 2.0 ** -25 * there
    assert ((mine - far).abs() <= 1e-9 * far)[there].all() and not mine[~there].any()


def test_the_batched_attention_knows_who_sees_a_nan():
    cache = [torch.ones(1, 1, 8, 16, dtype=torch.int8), torch.ones(1, 1, 8, 16, dtype=torch.int8), torch.ones(1, 1, 8), torch.ones(1, 1, 8)]
    cache[3][0, 0, 5] = float("nan")   # the first drafted token of three
    out, _ = forms.attention(torch.ones(1, 1, 3, 16), cache, torch.tensor([5]), torch.tensor([[-1, -1, 0]]))
    assert torch.isnan(out[0, 0, :, 0]).tolist() == [True, False, True] and ((out[0, 0, 1] - 1).abs() < 1e-12).all()

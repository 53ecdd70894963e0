"""Shapes for every form of the attention over a quantized cache (which one a call takes its plan says, csrc/cache_plan.h), and
the attention in 64 bits for whole batches at a time.  Test infrastructure."""
import math
import os
import subprocess
from typing import NamedTuple

import torch

import cache_oracle as oracle
from conftest import PKG, ROOT

PLAN = r"""
#include "cache_plan.h"
#include <cstdio>
int main() {
  long long s, h, hq, cap, n, dk;
  while(std::scanf("%lld %lld %lld %lld %lld %lld", &s, &h, &hq, &cap, &n, &dk) == 6) {
    const auto p = marian_hip::cache_attention_plan(s, h, hq, cap, n, dk);
    std::printf("%d %d %d %d %d %d %lld %lld\n", p.few, p.many, p.dp, p.qt, p.waves, p.least, (long long)p.target, (long long)p.row_tiles);
  }
}
"""


class Form(NamedTuple):
    kind: str    # "few", "some", "many": cache_attention_few_kernel, cache_attention_kernel, cache_attention_many_kernel
    dp: int      # values of a row as the kernel holds it
    rows: int    # that the form is made for: few: 1, 2, 4, 8; else sixteens to a wave
    waves: int


class Case(NamedTuple):
    form: Form
    S: int
    H: int
    G: int       # query heads to a head of keys
    n: int
    dk: int
    cap: int
    long: int    # positions that some sequences have
    tree: bool   # with a tree as well as with a chain
    split: bool  # the long sequences are in several parts


def form_of(few, many, dp, qt, waves):
    return Form("few" if few else "many" if many else "some", dp, few or qt, waves)


def plans(tmp_path, shapes):
    """what the plan says of (S, H, G, cap, n, dk): the form, and blocks of a part at the least, parts of all, row tiles"""
    (tmp_path / "plan.cpp").write_text(PLAN)
    exe = tmp_path / "plan"
    subprocess.run(["g++", "-std=c++17", "-I", os.path.join(ROOT, PKG, "csrc"), "-o", str(exe), str(tmp_path / "plan.cpp")], check=True)
    given = "\n".join("%d %d %d %d %d %d" % (s, h, h * g, cap, n, dk) for s, h, g, cap, n, dk in shapes)
    out = subprocess.run([str(exe)], input=given, capture_output=True, text=True, check=True).stdout
    rows = [tuple(map(int, line.split())) for line in out.splitlines()]
    return [(form_of(*r[:5]), *r[5:]) for r in rows]


# every form that the launchers hold, each for three types of activations and two of codes
FORMS = ([Form("few", dp, rows, w) for dp in (64, 128) for rows in (1, 2, 4, 8) for w in (4, 2, 1)] +
         [Form("some", dp, qt, w) for dp, qt in ((64, 1), (64, 2), (128, 1), (128, 2), (256, 1)) for w in (4, 2, 1)] +
         [Form("many", dp, qt, 4) for dp, qt in ((64, 1), (64, 2), (128, 1), (128, 2), (256, 1))])


def _cases():
    """Rows: the form's most and, of the same form, fewer; values: as many as it holds and fewer; entries by the number of waves;
    capacities on the side of the rule that the form is on, lengths of their own (most of them short)."""
    out = []
    entries = {4: [(3, 4), (5, 2)], 2: [(64, 32), (290, 8)], 1: [(256, 16), (64, 65)]}
    for f in FORMS:
        for turn in range(2):
            S, H = entries[f.waves][turn]
            dk = {64: (64, 48), 128: (128, 80), 256: (256, 144)}[f.dp][turn]
            if f.kind == "few":
                n, G = {1: [(1, 1), (1, 1)], 2: [(2, 1), (1, 2)], 4: [(2, 2), (3, 1)], 8: [(4, 2), (5, 1)]}[f.rows][turn]
                cap = max(300, 400000 // (S * H) + 1)
                long = min(cap - n, 20000 // f.waves if f.waves == 4 else cap - n - 1)
            elif f.kind == "some":
                n, G = {1: [(4, 4), (9, 1)], 2: [(8, 4), (17, 1)]}[f.rows][turn]
                if f.dp == 256 and turn:   # of rows this long the few rows, too
                    n, G = 1, 2
                cap = 3000 if f.waves == 4 else 330
                long = cap - n - 3
            elif f.rows == 1:
                n, G = [(64, 1), (7, 11)][turn]
                if f.dp == 256 and turn:
                    n, G = 70, 3
                S, H, cap = 3, 4, 2500
                long = cap - n - 3
            else:
                n, G = [(50, 4), (150, 3)][turn]   # (200 rows: the second 128 partly there; 450: four of them)
                S, H, cap = [(16, 4, 1800), (8, 4, 900)][turn]
                long = cap - n - 3
            out.append(Case(f, S, H, G, n, dk, cap, long, n > 1 and n <= 64, f.waves == 4 and not (f.kind == "many" and f.rows == 2 and turn == 1)))
    return out


CASES = _cases()


def lengths(c):
    """of the sequences: long for the second and the last one, 0, 1, ends inside and at blocks of 32 and 64, and short ones"""
    some = [0, 31, 1, 64, 33, 127, 5, 96, 128, 17]
    lens = [min(some[s % len(some)], c.cap - c.n) for s in range(c.S)]
    lens[1] = c.long
    lens[-1] = c.long - 37
    return lens


def parts(least, target, lens, n, cap):
    """into how many a sequence's positions are split"""
    if target == 1:
        return [1] * len(lens)
    blocks = [(min(l + n, cap) + 127) // 128 for l in lens]
    each = max(least, -(-sum(blocks) // target))
    return [max(1, -(-b // max(each, 4 if b <= 4 else 0, -(-b // 48)))) for b in blocks]


# ---- the attention in 64 bits, whole batches at a time ---------------------------------------------------------
def seen(parents, n, device):
    """[.., n, n]: whether a new token sees another"""
    if parents is None:
        return torch.ones(n, n, dtype=torch.bool, device=device).tril()[None]
    i = torch.arange(n, device=device)
    own = torch.eye(n, dtype=torch.float64, device=device)
    up = (parents.long()[:, :, None] == i) & (i < i[:, None])   # (a parent that is not before its child: the settled ones)
    reach = own + up.double()
    for _ in range(6):
        reach = (reach @ reach).clamp(max=1.0)
    return reach > 0


def weight_rounding(dtype, rows):
    """of a weight ahead of its product with a value: two float16 - the second one's half step, 2^-11 of what the first one leaves, which is
    up to 2^-11 of the weight - or one, of bfloat16 with more than 32 rows an entry"""
    return 2.0 ** -11 if dtype == torch.bfloat16 and rows > 32 else 2.0 ** -22


def attention(q, cache, lens, parents=None, counts=None, scale=None, rounding=None):
    """As cache_oracle.attention, in products of whole batches on the tensors' own device: -> (result, how far a kernel's may be).
    What a row sees of a NaN makes it NaN; a NaN that it does not see is not in it."""
    S, HQ, n, dk = q.shape
    k, v, ks, vs = cache
    H, cap, dev = k.shape[1], k.shape[2], q.device
    G, scale = HQ // H, scale or dk ** -0.5
    rounding = rounding or weight_rounding(q.dtype, G * n)
    out = torch.empty(q.shape, dtype=torch.float64, device=dev)
    tol = torch.empty_like(out)
    lens = lens.long().clamp(0, cap)
    m = torch.full_like(lens, n) if counts is None else counts.long().clamp(0, n)
    sees = seen(parents, n, dev).expand(S, n, n)
    # sequences of similar length together, in pieces that fit
    order = torch.argsort(lens).tolist()
    while order:
        pick = order[-max(1, min(len(order), (1 << 26) // (H * dk * (int(lens[order[-1]]) + n)))):]
        if len(pick) > 1 and int(lens[pick[-1]]) > 4 * int(lens[pick[0]]) + 200:   # (a long one by itself)
            pick = pick[-1:]
        order = order[:len(order) - len(pick)]
        at = torch.tensor(pick, device=dev)
        used = min(cap, int(lens[pick].max()) + n)
        Q = q[at].double().reshape(len(pick), H, G * n, dk)
        K, V = (t[at][:, :, :used].float().double() * s[at][:, :, :used, None].double() for t, s in ((k, ks), (v, vs)))
        vsc = vs[at][:, :, :used].double().abs()
        j = torch.arange(used, device=dev)[None] - lens[at][:, None]                     # [s, used]
        see = sees[at].gather(2, j.clamp(0, n - 1)[:, None].expand(-1, n, -1)) & (j >= 0)[:, None] & (j < n)[:, None]
        see = (see | (j < 0)[:, None])[:, None, None].expand(-1, H, G, -1, -1).reshape(len(pick), H, G * n, used)
        bad = torch.isnan(K).any(-1) | torch.isnan(V).any(-1)                             # [s, H, used]
        poisoned = (see & bad[:, :, None]).any(-1) | ~torch.isfinite(Q).all(-1)
        K, V, vsc, Q = (torch.nan_to_num(t, 0.0, 0.0, 0.0) for t in (K, V, vsc, Q))
        e = scale * (Q @ K.transpose(2, 3))
        hidden = ~see
        p = torch.softmax(e.masked_fill(hidden, -math.inf), -1).nan_to_num(0.0)
        got = p @ V
        # the bound of cache_oracle.bound, of what a row sees
        products = (scale * (Q.abs() @ K.abs().transpose(2, 3))).masked_fill(hidden, 0.0).amax(-1)
        count = see.sum(-1).double()
        d = products * (dk + 8) * 2.0 ** -23 + e.abs().masked_fill(hidden, 0.0).amax(-1) * 2.0 ** -21 + 2.0 ** -21 + count * 2.0 ** -24
        steps = see.double() @ (V.abs() / torch.where(vsc > 0, vsc, torch.ones_like(vsc))[..., None])
        widest = vsc[:, :, None].expand(-1, -1, G * n, -1).masked_fill(hidden, 0.0).amax(-1)
        smallest = 2.0 ** -25 / 2.0 ** 9 * widest[..., None] * steps
        far = (p @ V.abs()) * ((2 * d + rounding + count * 2.0 ** -24)[..., None]) + p.amax(-1)[..., None] * smallest * 16 + got.abs() * oracle.HALF[q.dtype]
        if q.dtype == torch.float16:   # (below 2^-14 its steps are 2^-24 whatever the value: half of one)
            far = far + 2.0 ** -25
        got = got.masked_fill(poisoned[..., None], math.nan).view(len(pick), HQ, n, dk)
        there = (torch.arange(n, device=dev) < m[at][:, None])[:, None, :, None]
        out[at] = torch.where(there, got, torch.zeros_like(got))
        tol[at] = torch.where(there, far.view(got.shape), torch.zeros_like(got))
    return out, tol

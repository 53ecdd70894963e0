"""How many bits weights have in the attention over pages: on the GPU its results against 64 bits, in every form, on inputs whose results are
next to zero; without a GPU, that the tolerance tells two terms of a weight from one."""
import pytest
import torch

import pages_weights
from conftest import load

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
HEADS, PAGE = 2, 16


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dk", [48, 64, 80, 128, 144, 256])
@pytest.mark.parametrize("positions", [25, 31, 40])
def test_one_term_would_be_seen(dtype, dk, positions):
    k, v = pages_weights.inputs(positions + dk, HEADS, positions, dk, dtype)
    want, tol = pages_weights.result(k, v), pages_weights.tolerance(k, v)
    assert ((pages_weights.emulated(k, v, 2) - want).abs() <= tol).all()
    over = (pages_weights.emulated(k, v, 1) - want).abs() / tol
    assert over.max() > 2 and (over > 1).any(-1).all()   # (in every head)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dk", [48, 64, 80, 128, 144, 256])
@pytest.mark.parametrize("group,n", [(1, 1), (5, 4), (8, 7), (16, 6)])
@pytest.mark.parametrize("positions", [25, 31, 40])
def test_weights(dtype, dk, group, n, positions):
    """The last of n tokens sees all positions; one wave has them, or two, or two halves"""
    pages = load("pages")
    k, v = pages_weights.inputs(positions + dk, HEADS, positions, dk, dtype)
    count = -(-positions // PAGE)
    kv = pages.newPagedCache(count, HEADS, PAGE, dk, dtype)
    slots = torch.arange(positions, dtype=torch.int32, device="cuda")[None]
    pages.writePages(kv, k[None].cuda(), v[None].cuda(), slots)
    q = torch.zeros(1, n, HEADS * group, dk, dtype=dtype, device="cuda").transpose(1, 2)
    q[..., 0] = 1
    table = torch.arange(count, dtype=torch.int32, device="cuda")[None]
    got = pages.AttentionOverPages(q, kv, table, torch.tensor([positions - n], dtype=torch.int32, device="cuda"), scale=1.0)
    got = got[0, :, -1].view(HEADS, group, dk).cpu().double()
    want, tol = pages_weights.result(k, v), pages_weights.tolerance(k, v)
    off = (got - want[:, None]).abs() / tol[:, None]
    assert (off <= 1).all(), off.max().item()

"""The embedding's gradient where most tokens of a large batch read one row: the
partial sums of thousands of windows meet in one place (sra.h k13)."""
from __future__ import annotations

import pytest
import torch

import lm_reference as ref
import srfl_amd.lm as lm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("share", [0.5, 0.95, 1.0])
@pytest.mark.parametrize("E", [9, 520])
def test_a_row_of_most_tokens(E, share):
    T, V = 262147, 1000
    g = torch.Generator().manual_seed(E)
    ids = torch.where(torch.rand(T, generator=g) < share, torch.full((T,), 7), torch.randint(0, V, (T,), generator=g))
    dy = torch.randint(-3, 4, (T, E), generator=g).to(torch.bfloat16).cuda()
    ids = ids.cuda()
    # whole numbers below 2^24 add up without rounding in any order
    want, _ = ref.embed_grad(dy, ids, 1, V, None, None, 1.0)
    grad = lm.embed_grad(dy, ids, torch.full((V, E), 7.0, device="cuda"))
    assert torch.equal(grad.cpu().double(), want[0])
    start = torch.randint(0, 9, (V, E), generator=g).float().cuda()
    added = lm.embed_grad(dy, ids, start.clone(), accumulate=True)
    assert torch.equal(added.cpu().double(), want[0] + ref.d(start))
    left = lm.embed_grad(dy, ids, torch.empty(V, E, device="cuda"), padding_idx=7)
    want[0][7] = 0
    assert torch.equal(left.cpu().double(), want[0])

"""engine.row_fault_count after slots outside the clients' matrices: one a token
and call, whatever the launches look like."""
from __future__ import annotations

import pytest
import torch

import srfl_amd.engine as engine
import srfl_amd.lm as lm

pytestmark = pytest.mark.gpu


def rand(*shape, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(0)).to(dtype).cuda()


def seg(offsets, slots):
    return torch.tensor(offsets, dtype=torch.int64).cuda(), torch.tensor(slots, dtype=torch.int32).cuda()


def counted(f):
    engine.row_fault_count(reset=True)
    f()
    return engine.row_fault_count(reset=True)


@pytest.mark.parametrize("T,E", [(40, 16), (5000, 8), (40, 300)])
def test_embedding(T, E):
    offsets, slots = [1, 9, 9, 20, T], [0, 7, -3, 1]         # the empty segment of slot 7 holds no token
    o, s = seg(offsets, slots)
    table, ids, dy = rand(2, 6, E), (torch.arange(T) % 6).cuda(), rand(T, E)
    assert counted(lambda: lm.embed(table, ids, o, s)) == 11
    assert counted(lambda: lm.embed_grad(dy, ids, torch.empty_like(table), o, s)) == 11
    ids[12] = 99                                            # in a bad slot: counted already
    ids[25] = 99
    assert counted(lambda: lm.embed(table, ids, o, s)) == 12
    assert counted(lambda: lm.embed_grad(dy, ids, torch.empty_like(table), o, s)) == 12


@pytest.mark.parametrize("T,K,M,r,segments", [
    (40, 32, 48, 4, 1), (700, 32, 48, 4, 1),                # tiles of 64 tokens
    (200, 32, 48, 4, 100),                                  # tiles of 16
    (300, 1040, 2050, 16, 1), (33, 9000, 300, 33, 20),      # parts of the width, several column blocks
    (50, 5, 40, 3, 1), (50, 40, 5, 3, 1), (50, 5, 5, 3, 30),    # element by element
])
def test_adapters(T, K, M, r, segments):
    cuts = sorted(set([0, 2] + [2 + (T - 5) * i // segments for i in range(1, segments + 1)]))
    slots = [(0, 5, 1, -2)[i % 4] for i in range(len(cuts) - 1)] + [9]       # the last one is empty
    offsets = cuts + [cuts[-1]]
    bad = sum(b - a for a, b, c in zip(offsets, offsets[1:], slots) if c not in (-1, 0, 1))
    assert bad > 0
    o, s = seg(offsets, slots)
    x, base, A, B, dy = rand(T, K), rand(T, M), rand(2, r, K), rand(2, M, r), rand(T, M)
    assert counted(lambda: lm.adapter_apply(base, x, A, B, o, s)) == bad
    _, h = lm.adapter_apply(base, x, A, B, o, s, hidden=True)
    for hidden in (None, h):
        for gx, ga, gb in ((True, True, True), (True, False, False), (False, True, False), (False, False, True),
                           (True, False, True)):
            assert counted(lambda: lm.adapter_grad(dy, x, A, B, o, s, hidden=hidden, grad_x=gx, grad_A=ga,
                                                   grad_B=gb)) == bad, (hidden is None, gx, ga, gb)
    assert counted(lambda: lm.adapter_grad(dy, x, A, B, o, s, grad_x=False, grad_A=False, grad_B=False)) == 0

"""Adapters with float32 activations (sra.h k12): they run on the float32 matrix
units, so nothing but float32 summation may show: no term of a product is left
out, and operands in two bf16 terms (2^-18 each) would fail the narrow cases."""
from __future__ import annotations

import pytest
import torch

import lm_reference as ref
import srfl_amd.lm as lm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,K,M,r,offsets,slots", [
    (9, 8, 8, 2, [0, 5, 9], [1, 0]), (70, 16, 9, 1, [0, 70], [0]), (1, 64, 64, 8, [0, 1], [0]), (17, 100, 33, 5, [0, 16, 17], [1, 0]), (65, 320, 192, 17, [0, 65], [0]),
    (200, 520, 260, 64, [0, 150, 200], [1, 0]), (40, 1031, 7, 3, [0, 20, 40], [0, 1]),
    (100, 48, 80, 16, list(range(0, 101, 2)), [i % 3 for i in range(50)]),
])
def test_every_bit_of_the_products(T, K, M, r, offsets, slots, monkeypatch):
    monkeypatch.setattr(ref, "PROD", 0.0)
    g = torch.Generator().manual_seed(T)
    n = max(slots) + 1
    x, base, dy, dxb = (torch.randn(T, w, generator=g).cuda() for w in (K, M, M, K))
    A, B = (torch.randn(n, *q, generator=g).cuda() for q in ((r, K), (M, r)))
    o, s = torch.tensor(offsets).cuda(), torch.tensor(slots, dtype=torch.int32).cuda()
    want = ref.adapter(base, x, A, B, offsets, slots, 0.7, torch.float32, dy, dxb)
    y, h = lm.adapter_apply(base, x, A, B, o, s, 0.7, hidden=True)
    ref.within("out", y, *want["out"])
    for hidden in (h, None):
        got = lm.adapter_grad(dy, x, A, B, o, s, 0.7, hidden=hidden, base_grad=dxb)
        for name, t in zip(("dx", "dA", "dB"), got):
            ref.within(name, t, *want[name])


def test_the_bound_tells_two_terms_apart(monkeypatch):
    """Products of operands in two bf16 terms, summed in 64 bits, are beyond the bound
    of the narrowest case."""
    monkeypatch.setattr(ref, "PROD", 0.0)
    g = torch.Generator().manual_seed(1)
    x, A = torch.randn(64, 8, generator=g), torch.randn(8, 5, generator=g)

    def two(t):
        hi = t.bfloat16().float()
        return (hi + (t - hi).bfloat16().float()).double()

    v, e = ref.product(x.double(), torch.zeros(64, 8).double(), A.double(), torch.zeros(8, 5).double())
    assert ((two(x) @ two(A) - v).abs() > e).any()

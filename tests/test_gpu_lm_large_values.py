"""Adapters (sra.h k12) with finite operands next to float32's largest value, which
no bf16 number is near: the nearest one is infinite."""
from __future__ import annotations

import pytest
import torch

import lm_reference as ref
import srfl_amd.lm as lm

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
TOP = torch.finfo(torch.float32).max


def rand(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T,K,M,r,offsets", [(3, 64, 40, 4, [0, 1, 3]), (150, 136, 72, 20, [0, 80, 150]),
                                             (64, 2056, 48, 8, [0, 30, 64])])
def test_weights_and_hidden_values(T, K, M, r, offsets, dtype):
    """One weight of A, one of B, and hidden values and z beside the largest float32,
    each against small values on the other side, so that every result is finite."""
    o, s = torch.tensor(offsets).cuda(), torch.tensor([1, 0], dtype=torch.int32).cuda()
    dt = DT[dtype]
    tiny = 2.0 ** -14                                        # normal in fp16 too
    A, B = rand(2, r, K) * 0.1, rand(2, M, r, seed=1) * 0.1
    x, base, dy = rand(T, K, seed=2), rand(T, M, seed=3), rand(T, M, seed=4)

    def check(name):
        args = [t.cuda() for t in (A, B)]
        acts = [t.to(dt).cuda() for t in (x, base, dy)]
        want = ref.adapter(acts[1], acts[0], *args, offsets, [1, 0], 2.0 ** -20, dt, acts[2])
        y, h = lm.adapter_apply(acts[1], acts[0], *args, o, s, 2.0 ** -20, hidden=True)
        dx, dA, dB = lm.adapter_grad(acts[2], acts[0], *args, o, s, 2.0 ** -20, hidden=h)
        assert torch.isfinite(h).all(), name
        for key, got in (("dA", dA), ("dB", dB)):
            assert torch.isfinite(want[key][0]).all()
            ref.within(name + " " + key, got, *want[key])
        # out and dx leave fp16's range where the formula does
        for key, got in (("out", y), ("dx", dx)):
            v, e = want[key]
            # below the type's normal range a rounding is off by half its smallest step (fp16 2^-25), not by
            # half a step of the value, which is all that the oracle's bound holds
            e = e + torch.finfo(dt).tiny * torch.finfo(dt).eps / 2
            inside = v.abs() + e < torch.finfo(dt).max
            assert torch.isfinite(ref.d(got)[inside]).all() and not torch.isnan(got).any(), name + " " + key
            ref.within(name + " " + key, torch.where(inside, ref.d(got), v), v, e)

    A[1, 1, 3] = TOP                                         # x stays small beside it
    x[:, 3] = tiny * torch.sign(x[:, 3])
    check("a weight of A")
    A[1, 1, 3] = 0.1
    B[0, 5, 2] = -TOP
    A[0, 2] *= 2.0 ** -30                                    # hidden values of rank 2 stay small
    dy[:, 5] = tiny * torch.sign(dy[:, 5])
    check("a weight of B")


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_hidden_values(dtype):
    """Hidden values of 3.4e38 times weights of 1e-36.  (Sums that reach float32's
    largest value from below, like 2 * 1.7e38, may pass it on their way: the nearest
    bf16 of 1.7e38 lies above it.)"""
    dt = DT[dtype]
    T, K, M, r = 20, 64, 48, 4
    o, s = torch.tensor([0, T]).cuda(), torch.zeros(1, dtype=torch.int32).cuda()
    A = torch.zeros(1, r, K)
    A[0, :, 0] = TOP
    x = torch.zeros(T, K)
    x[:, 0] = 1.0
    B = rand(1, M, r).abs() * 1e-36
    acts = [x.to(dt).cuda(), A.cuda(), B.cuda()]
    y, h = lm.adapter_apply(None, *acts, o, s, hidden=True)
    assert (h == TOP).all()
    want = ref.adapter(None, x.to(dt), A, B, [0, T], [0], 1.0, dt)
    ref.within("out", y, *want["out"])
    dy = (torch.ones(T, M) * 2.0 ** -14).to(dt)
    _, _, dB = lm.adapter_grad(dy.cuda(), *acts, o, s, hidden=h, grad_x=False, grad_A=False, scale=2.0 ** -10)
    want = ref.adapter(None, x.to(dt), A, B, [0, T], [0], 2.0 ** -10, dt, dy)
    ref.within("dB", dB, *want["dB"])


def test_infinite_operands_stay_infinite_or_nan():
    T, K, M, r = 4, 64, 48, 4
    o, s = torch.tensor([0, T]).cuda(), torch.zeros(1, dtype=torch.int32).cuda()
    A, B = rand(1, r, K).abs() + 0.1, rand(1, M, r).abs() + 0.1
    x = (rand(T, K).abs() + 0.5).bfloat16()
    for bad in (float("inf"), float("nan")):
        A2, B2 = A.clone(), B.clone()
        A2[0, 1, 3] = bad
        y, h = lm.adapter_apply(None, x.cuda(), A2.cuda(), B.cuda(), o, s, hidden=True)
        assert not torch.isfinite(h[:, 1]).any() and torch.isfinite(h[:, [0, 2, 3]]).all() and not torch.isfinite(y).any()
        B2[0, 7, 2] = bad
        y = lm.adapter_apply(None, x.cuda(), A.cuda(), B2.cuda(), o, s)
        keep = torch.arange(M) != 7
        assert not torch.isfinite(y[:, 7]).any() and torch.isfinite(y[:, keep]).all()

"""Results written into the caller's tensors raise their versions, so autograd
notices that a tensor it saved was overwritten."""
from __future__ import annotations

import pytest
import torch

import srfl_amd.lm as lm
import srfl_amd.store as store

pytestmark = pytest.mark.gpu


def rand(*shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(0)).cuda()


def seg(T):
    return torch.tensor([0, T]).cuda(), torch.zeros(1, dtype=torch.int32).cuda()


def calls():
    T, K, M, r, V = 6, 16, 24, 2, 10
    o, s = seg(T)
    x, base, A, B, dy, dxb = rand(T, K), rand(T, M), rand(1, r, K), rand(1, M, r), rand(T, M), rand(T, K)
    logits, t, gl, ids = rand(T, V), torch.arange(T).cuda(), rand(T), (torch.arange(T) % 5).cuda()
    lse = lm.token_logprobs(logits, t).lse
    out, dx, dA, dB, g = (torch.empty_like(q) for q in (base, x, A, B, logits))
    emb, table = torch.empty(T, 4, device="cuda"), rand(5, 4)
    return {
        "apply": ([out], lambda: lm.adapter_apply(base, x, A, B, o, s, out=out)),
        "apply in place": ([base], lambda: lm.adapter_apply(base, x, A, B, o, s, out=base)),
        "grad": ([dx, dA, dB], lambda: lm.adapter_grad(dy, x, A, B, o, s, grad_x=dx, grad_A=dA, grad_B=dB)),
        "grad in place": ([dxb], lambda: lm.adapter_grad(dy, x, A, B, o, s, base_grad=dxb, grad_x=dxb)),
        "embed": ([emb], lambda: lm.embed(table, ids, out=emb)),
        "embed_grad": ([table], lambda: lm.embed_grad(emb, ids, table)),
        "logprobs": ([g], lambda: lm.token_logprobs_and_grad(logits, t, gl, out=g)),
        "logprobs grad": ([g], lambda: lm.token_logprobs_grad(logits, t, lse, gl, out=g)),
        "logprobs in place": ([logits], lambda: lm.token_logprobs_and_grad(logits, t, gl, out=logits)),
    }


@pytest.mark.parametrize("name", ["apply", "apply in place", "grad", "grad in place", "embed", "embed_grad", "logprobs",
                                  "logprobs grad", "logprobs in place"])
def test_versions_rise(name):
    written, call = calls()[name]
    before = [t._version for t in written]
    call()
    assert all(t._version > b for t, b in zip(written, before))


def test_inputs_keep_their_versions():
    T = 6
    o, s = seg(T)
    ins = [rand(T, 24), rand(T, 16), rand(1, 2, 16), rand(1, 24, 2)]
    before = [t._version for t in ins]
    lm.adapter_apply(*ins, o, s)
    lm.adapter_grad(ins[0], *ins[1:], o, s, base_grad=ins[1])
    assert [t._version for t in ins] == before


def test_a_view_of_a_saved_tensor():
    """The buffer's other views share its version."""
    T = 6
    o, s = seg(T)
    buf = rand(T, 30)
    w = rand(30).requires_grad_()
    loss = (buf * w).sum()                                   # saves buf
    lm.adapter_apply(None, rand(T, 16), rand(1, 2, 16), rand(1, 24, 2), o, s, out=buf[:, 3:27])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_inference_tensors_have_none():
    T = 6
    o, s = seg(T)
    with torch.inference_mode():
        out = torch.empty(T, 24, device="cuda")
        lm.adapter_apply(None, rand(T, 16), rand(1, 2, 16), rand(1, 24, 2), o, s, out=out)
    assert torch.isfinite(out).all()


def test_a_bank_that_records():
    """Its rows go back to the snapshot."""
    params = [rand(5, 4), rand(3)]
    S = store.ClientStore(params, 3)
    S.snapshot()
    bank = store.ClientBank(S, 2)
    bank.load([2, 0])
    bank.G.fill_(1.0)
    bank.step(0.5)
    w = rand(2, 5, 4).requires_grad_()
    loss = (bank.param(0) * w).sum()                         # saves the rows
    bank.record()
    assert torch.equal(bank.param(0)[0], params[0])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()

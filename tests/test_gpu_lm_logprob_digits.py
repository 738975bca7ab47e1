"""Log probabilities and gradients whose digits do not depend on how large the
logits are (sra.h k14): only differences of logits enter.

Bounds.  With d = x - max, s = sum exp(d) has the relative error rel of its
terms (2 |d| + 4 roundings each, weighted) and of its summation, so log s is off
by rel + 2 U |log s|.  max + log s is held as two floats without a further
error, and x minus them is exact where the two are within a factor of two of one
another and else a rounding of a difference that is as large as the result: 3 U of
the result with the second subtraction.  Neither |x| nor |lse| appears.  A 16-bit gradient may
leave out what the rounding of an lse below 16 left: 2^-21 of p."""
from __future__ import annotations

import pytest
import torch

import lm_reference as ref
import srfl_amd.lm as lm

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
U = ref.U


def exact(x, t):
    x = ref.d(x)
    V = x.shape[1]
    steps = V / 64 + 32
    m = x.max(1, keepdim=True).values
    dd = x - m
    p = torch.exp(dd)
    s = p.sum(1, keepdim=True)
    p, ls = p / s, torch.log(s)
    logp = dd - ls
    far = torch.where(p > 0, dd, torch.zeros_like(dd))
    a1, a2 = (p * far.abs()).sum(1, keepdim=True), (p * far * far).sum(1, keepdim=True)
    ent = ls - (p * far).sum(1, keepdim=True)
    rel = U * (2 * a1 + 4 + steps)
    e_ls = rel + 2 * U * ls.abs()
    e_ent = 2 * rel + U * (2 * a2 + (steps + 8) * a1 + 2 * ls.abs() + 2 * ent.abs()) + rel * a1
    return dict(x=x, t=t.cpu(), p=p, logp=logp, e_ls=e_ls, ent=ent, e_ent=e_ent, e_logp=e_ls + 3 * U * logp.abs())


def at_target(w):
    t = w["t"][:, None]
    return w["logp"].gather(1, t).squeeze(1), w["e_logp"].gather(1, t).squeeze(1)


def gradient(w, gl, ge, dtype):
    p, l = w["p"], w["logp"]
    l = torch.where(p > 0, l, torch.zeros_like(l))
    gl = ref.d(gl)[:, None]
    ep = p * (w["e_ls"] + U * (5 * l.abs() + 4) + (2.0 ** -21 if dtype != torch.float32 else 0.0))
    g, err = -gl * p, gl.abs() * ep + 3 * U * gl.abs() * p
    if ge is not None:
        ge = ref.d(ge)[:, None]
        f = l + w["ent"]
        g = g - ge * p * f
        err = err + ge.abs() * (ep * f.abs() + p * (U * (3 * l.abs() + 4 * f.abs()) + w["e_ls"] + w["e_ent"])) \
            + U * (gl * p).abs()
    g = g.scatter_add(1, w["t"][:, None], gl)
    err = err + 2 * U * (g.abs() + gl.abs())
    tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    return g, err + ref.half_step(dtype) * (g.abs() + err) + tiny + 2.0 ** -126 * (gl.abs() + 1)


def rows(V, dtype, seed=0):
    """Rows whose logits sit anywhere in the type's range, and their targets."""
    g = torch.Generator().manual_seed(seed)
    big = 30000.0 if dtype != torch.float16 else 20000.0
    low = torch.finfo(dtype).min
    x = torch.randn(10, V, generator=g) * 3
    t = torch.randint(0, V, (10,), generator=g)
    x[1] += big
    x[2] -= big
    x[3] += 1000.0
    x[4] = 6.0 + x[4].clamp(max=0) - 14.0                # a target that is all but certain
    x[4, t[4]] = 20.0
    x[5] = low                                           # a mask of the type's lowest value that leaves nothing
    x[6] = -low
    x[7] = low                                           # one that leaves a few
    x[7, ::3] = torch.randn(len(x[7, ::3]), generator=g)
    x[8] = x[8] * 1e-3 + big
    x[9] = 0.0
    return x.to(dtype).cuda(), t.cuda()


def weights(seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(10, generator=g).cuda(), torch.randn(10, generator=g).cuda()


SIZES = [5, 64, 777, 2048, 4099, 40001, 70001]


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("V", SIZES)
def test_log_probabilities(V, dtype):
    x, t = rows(V, DT[dtype], V)
    w = exact(x, t)
    want, bound = at_target(w)
    res = lm.token_logprobs(x, t, top=3, entropy=True)
    ref.within("logp", res.logp, want, bound)
    ref.within("entropy", res.entropy, w["ent"].squeeze(1), w["e_ent"].squeeze(1))
    ids = res.top_ids.cpu()
    ref.within("top_logp", res.top_logp, w["logp"].gather(1, ids), w["e_logp"].gather(1, ids))


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("V", SIZES)
def test_gradient_in_one_pass(V, dtype):
    x, t = rows(V, DT[dtype], V)
    w = exact(x, t)
    gl, ge = weights(V)
    for gent in (None, ge):
        res, grad = lm.token_logprobs_and_grad(x, t, gl, gent, entropy=True)
        ref.within("logp", res.logp, *at_target(w))
        ref.within("grad", grad, *gradient(w, gl, gent, DT[dtype]))


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("V", SIZES)
def test_gradient_from_a_forward_pass(V, dtype):
    x, t = rows(V, DT[dtype], V)
    w = exact(x, t)
    gl, ge = weights(V)
    res = lm.token_logprobs(x, t, entropy=True)
    for gent in (None, ge):
        grad = lm.token_logprobs_grad(x, t, res.lse, gl, res.entropy, gent, lse_rest=res.lse_rest)
        ref.within("grad", grad, *gradient(w, gl, gent, DT[dtype]))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_gradient_by_autograd(dtype):
    x, t = rows(777, DT[dtype])
    w = exact(x, t)
    gl, ge = weights(3)
    leaf = x.clone().requires_grad_()
    logp, ent = lm.token_logp(leaf, t)
    (logp * gl + ent * ge).sum().backward()
    ref.within("grad", leaf.grad, *gradient(w, gl, ge, DT[dtype]))


def test_a_common_offset_changes_nothing():
    """Logits on a grid that an offset of 2^15 keeps: the same differences, so the same numbers."""
    g = torch.Generator().manual_seed(2)
    x = (torch.randn(6, 5003, generator=g) * 4 * 256).round().div(256).cuda()
    t = torch.randint(0, 5003, (6,), generator=g).cuda()
    gl = torch.ones(6, device="cuda")
    near, gnear = lm.token_logprobs_and_grad(x, t, gl)
    far, gfar = lm.token_logprobs_and_grad(x + 32768.0, t, gl)
    w = exact(x, t)
    want, bound = at_target(w)
    ref.within("near", near.logp, want, bound)
    ref.within("far", far.logp, want, bound)
    value, err = gradient(w, gl, None, torch.float32)
    ref.within("gradient near", gnear, value, err)
    ref.within("gradient far", gfar, value, err)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_entries_without_the_rest(dtype):
    """The C entries that know lse alone: the same numbers but the rest."""
    from srfl_amd import _lib
    R, V = 10, 5003
    x, t = rows(V, DT[dtype], 4)
    gl, _ = weights(4)
    code, stream = {"fp32": 0, "bf16": 1}[dtype], torch.cuda.current_stream().cuda_stream
    res, grad = lm.token_logprobs_and_grad(x, t, gl, top=2)
    logp, lse = torch.empty(2, R, device="cuda").unbind(0)
    tl, ti, g = torch.empty_like(res.top_logp), torch.empty_like(res.top_ids), torch.empty_like(x)
    _lib.call("sra_token_logprobs", x.data_ptr(), V, code, t.data_ptr(), R, V, -100, 2, logp.data_ptr(), None,
              lse.data_ptr(), tl.data_ptr(), ti.data_ptr(), gl.data_ptr(), None, g.data_ptr(), V, stream)
    for a, b in ((logp, res.logp), (lse, res.lse), (tl, res.top_logp), (ti, res.top_ids), (g, grad)):
        assert torch.equal(a, b)
    _lib.call("sra_token_logprobs_grad", x.data_ptr(), V, code, t.data_ptr(), R, V, -100, lse.data_ptr(), None,
              gl.data_ptr(), None, g.data_ptr(), V, stream)
    assert torch.equal(g, lm.token_logprobs_grad(x, t, lse, gl))

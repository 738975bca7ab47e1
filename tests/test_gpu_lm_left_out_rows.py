"""Rows that a loss leaves out (ignored or bad target, weight zero) get a zero
gradient of the logits whatever they hold (sra.h k14)."""
from __future__ import annotations

import pytest
import torch

import srfl_amd.engine as engine
import srfl_amd.lm as lm

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
INF, NAN = float("inf"), float("nan")


def make(V, dtype):
    g = torch.Generator().manual_seed(V)
    x = torch.randn(9, V, generator=g)
    for r in (0, 3, 6):
        x[r] = -INF
        x[r + 1, V // 2] = NAN
        x[r + 2, V - 1] = INF
    t = torch.randint(0, V, (9,), generator=g)
    t[:3] = -100                                            # ignored
    t[3:6] = torch.tensor([V, -1, V + 5])                   # outside the vocabulary
    gl = torch.full((9,), -0.5)
    gl[6:] = 0.0                                            # weight zero
    return x.to(dtype).cuda(), t.cuda(), gl.cuda()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("V", [3, 500, 2049, 5003, 40001, 70001])
def test_gradient_is_zero(V, dtype):
    x, t, gl = make(V, DT[dtype])
    res, g = lm.token_logprobs_and_grad(x, t, gl, entropy=True)
    assert not g.any()
    assert not res.logp[:3].any() and torch.isnan(res.logp[3:]).all()
    assert not lm.token_logprobs_grad(x, t, res.lse, gl).any()
    zero = torch.zeros(9, device="cuda")
    y = x.clone()
    lm.token_logprobs_and_grad(y, t, gl, zero, out=y)
    assert not y.any()
    y = x.clone()
    lm.token_logprobs_grad(y, t, res.lse, gl, res.entropy, zero, out=y)
    assert not y.any()
    engine.row_fault_count(reset=True)


def test_rows_that_count_keep_their_nan():
    x, t, gl = make(700, torch.float32)
    t, gl = torch.zeros_like(t), torch.ones_like(gl)
    res, g = lm.token_logprobs_and_grad(x, t, gl)
    assert torch.isnan(g).any(1).all() and torch.isnan(lm.token_logprobs_grad(x, t, res.lse, gl)).any(1).all()


def test_a_padding_row_leaves_the_other_tokens_alone():
    """The product with the output layer's weight, as a training step goes on."""
    x, t, gl = make(300, torch.float32)
    leaf = x.clone().requires_grad_()
    logp, _ = lm.token_logp(leaf, t)
    torch.where(t == -100, torch.zeros_like(logp), logp)[:3].sum().backward()
    assert not (leaf.grad @ torch.ones(300, 8, device="cuda")).any()
    engine.row_fault_count(reset=True)

"""Log probabilities of given tokens, entropy, top alternatives and the logits'
gradient (sra.h k14)."""
from __future__ import annotations

import pytest
import torch

import lm_reference as ref
import srfl_amd.engine as engine
import srfl_amd.lm as lm

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
INF = float("inf")


def make(R, V, dtype, seed=0, std=3.0, pad=0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(R, V + pad, generator=g) * std).to(dtype).cuda()[:, :V]
    return x, torch.randint(0, V, (R,), generator=g).cuda()


def best(x, k):
    """The k largest, descending, the lowest index first among equals, NaN on top."""
    v = x.float().cpu()
    key = torch.where(torch.isnan(v), torch.full_like(v, INF), v) + 0.0
    nan = torch.isnan(v).to(torch.float64)
    out = []
    for r in range(v.shape[0]):
        out.append(sorted(range(v.shape[1]), key=lambda i: (-nan[r, i].item(), -key[r, i].item(), i))[:k])
    return torch.tensor(out).view(v.shape[0], k)


def check(x, t, top, dtype, seed=0):
    R, V = x.shape
    res = lm.token_logprobs(x, t, top=top, entropy=True)
    want = ref.logprobs(x, t)
    ref.within("lse", res.lse, want["lse"], want["e_lse"])
    ref.within("logp", res.logp, want["logp"], want["e_logp"])
    ref.within("entropy", res.entropy, want["ent"], want["e_ent"])
    if top:
        ids = best(x, top)
        assert torch.equal(res.top_ids.cpu(), ids)
        tl = want["x"].gather(1, ids) - want["lse"][:, None]
        ref.within("top_logp", res.top_logp, tl, want["e_lse"][:, None] + ref.U * (2 * tl.abs() + 1))
    g = torch.Generator().manual_seed(seed + 50)
    gl, ge = torch.randn(R, generator=g).cuda(), torch.randn(R, generator=g).cuda()
    for gent in (None, ge):
        wg, bound = ref.logits_grad(want, t, gl, gent, dtype)
        both, grad = lm.token_logprobs_and_grad(x, t, gl, gent, top=top, entropy=True)
        ref.within("grad", grad, wg, bound)
        # another number of waves may sum the row in another order
        ref.within("lse with grad", both.lse, want["lse"], want["e_lse"])
        ref.within("logp with grad", both.logp, want["logp"], want["e_logp"])
        ref.within("entropy with grad", both.entropy, want["ent"], want["e_ent"])
        assert torch.equal(both.top_ids, res.top_ids)
        grad2 = lm.token_logprobs_grad(x, t, res.lse, gl, res.entropy, gent)
        ref.within("grad from lse", grad2, wg, bound)
    return res


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("R,V,top", [(1, 1, 1), (1, 2, 2), (3, 7, 5), (5, 64, 32), (4, 65, 0), (130, 10, 3),
                                     (3, 511, 1), (2, 512, 20), (2, 513, 20), (3, 2055, 7), (9, 5003, 4),
                                     (1, 40001, 5), (2, 20000, 32), (2, 70001, 3), (1030, 2100, 2)])
def test_rows(R, V, top, dtype):
    x, t = make(R, V, DT[dtype])
    check(x, t, min(top, V), DT[dtype])


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_strided_rows_and_odd_starts(dtype):
    for pad in (1, 3, 8):
        x, t = make(6, 1001, DT[dtype], pad=pad)
        check(x, t, 4, DT[dtype])
    x, t = make(6, 1009, DT[dtype])
    check(x[:, 3:1004], t.clamp(max=1000), 4, DT[dtype])
    check(x[:, ::2], t // 2, 4, DT[dtype])                   # strided columns are copied


def test_ties_take_the_lowest_index():
    x = torch.zeros(4, 3000, device="cuda")
    x[1] = 5.0
    x[2, ::7] = 2.0
    x[3, 1500:] = -0.0                                        # -0 equals +0
    t = torch.zeros(4, dtype=torch.int64, device="cuda")
    res = check(x, t, 9, torch.float32)
    assert res.top_ids[0].tolist() == list(range(9)) and res.top_ids[2].tolist() == [7 * i for i in range(9)]
    x, t = make(20, 5000, torch.bfloat16, std=0.3)            # few distinct values
    check(x, t, 32, torch.bfloat16)


@pytest.mark.parametrize("order", ["ascending", "descending", "zigzag"])
def test_sorted_rows(order):
    v = torch.linspace(-20, 20, 9000)
    if order == "descending":
        v = v.flip(0)
    elif order == "zigzag":
        v = torch.stack([v, -v], 1).flatten()
    x = v.repeat(2, 1).cuda()
    check(x, torch.tensor([0, 5000]).cuda(), 32, torch.float32)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_masked_logits(dtype):
    x, t = make(8, 700, DT[dtype])
    low = torch.finfo(DT[dtype]).min
    x[0, 100:] = -INF
    x[1, :699] = -INF
    x[2, ::2] = low
    x[3] = low                                                # one value everywhere: uniform
    x[4, 10:20] = -INF
    t[0], t[1], t[2], t[4] = 5, 699, 1, 12
    res = check(x, t, 5, DT[dtype])
    assert res.logp[1] == 0 and res.entropy[1] == 0 and res.logp[4] == -INF
    assert res.top_ids[1].tolist() == [699, 0, 1, 2, 3]


def test_nan_inf_and_empty_rows():
    x, t = make(5, 900, torch.float32)
    x[0] = -INF
    x[1, 450] = INF
    x[2, 7] = float("nan")
    x[3, 899] = float("nan")
    t[:] = 3
    res = lm.token_logprobs(x, t, top=3, entropy=True)
    for v in (res.logp, res.entropy, res.lse[1:]):
        assert torch.isnan(v[:3]).all()
    assert torch.isnan(res.logp[:4]).all() and torch.isfinite(res.logp[4])
    assert res.top_ids[0].tolist() == [0, 1, 2] and res.top_ids[1, 0] == 450
    assert res.top_ids[2, 0] == 7 and res.top_ids[3, 0] == 899
    _, g = lm.token_logprobs_and_grad(x, t, torch.ones(5, device="cuda"))
    assert torch.isnan(g[:4]).any(1).all() and torch.isfinite(g[4]).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_large_logits_do_not_overflow(dtype):
    x, t = make(3, 300, DT[dtype], std=1.0)
    x[0] += 30000.0
    x[1] -= 30000.0
    x[2, 5] = 1.0e30
    check(x, t, 3, DT[dtype])


def test_ignored_and_bad_targets():
    x, t = make(6, 100, torch.bfloat16)
    t[1] = t[4] = -100
    gl = torch.ones(6, device="cuda")
    res, g = lm.token_logprobs_and_grad(x, t, gl)
    assert res.logp[1] == 0 and res.logp[4] == 0 and not g[[1, 4]].any() and g[0].any()
    other = lm.token_logprobs(x, torch.where(t == -100, 7, t), ignore_index=7)
    assert other.logp[1] == 0
    engine.row_fault_count(reset=True)
    t[2], t[3] = 100, -3
    res, g = lm.token_logprobs_and_grad(x, t, gl)
    assert engine.row_fault_count(reset=True) == 2
    assert torch.isnan(res.logp[[2, 3]]).all() and torch.isfinite(res.lse).all() and not g[[2, 3]].any()
    g = lm.token_logprobs_grad(x, t, res.lse, gl)
    assert engine.row_fault_count(reset=True) == 2 and not g[[2, 3]].any()


@pytest.mark.parametrize("V", [10, 777, 4100, 40001, 66001])
def test_gradient_in_place(V):
    x, t = make(7, V, torch.bfloat16)
    gl, ge = torch.full((7,), -0.25, device="cuda"), torch.full((7,), 0.5, device="cuda")
    res, want = lm.token_logprobs_and_grad(x, t, gl, ge, entropy=True)
    y = x.clone()
    res2, got = lm.token_logprobs_and_grad(y, t, gl, ge, out=y)
    assert got.data_ptr() == y.data_ptr() and torch.equal(y, want) and torch.equal(res2.logp, res.logp)
    y = x.clone()
    lm.token_logprobs_grad(y, t, res.lse, gl, res.entropy, ge, out=y)
    # the same formula with the same lse and entropy
    assert torch.equal(y, want)
    wide = torch.full((7, V + 3), 7.0, dtype=torch.bfloat16, device="cuda")
    lm.token_logprobs_and_grad(x, t, gl, ge, out=wide[:, 1:V + 1])
    assert torch.equal(wide[:, 1:V + 1], want) and (wide[:, 0] == 7).all() and (wide[:, V + 1:] == 7).all()


def test_graph_replays():
    x, t = make(40, 3001, torch.bfloat16)
    gl = torch.full((40,), -1 / 40, device="cuda")
    lm.token_logprobs_and_grad(x, t, gl, top=3, entropy=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res, g = lm.token_logprobs_and_grad(x, t, gl, top=3, entropy=True)
    for i in range(4):
        nx, nt = make(40, 3001, torch.bfloat16, seed=i)
        x.copy_(nx)
        t.copy_(nt)
        graph.replay()
        torch.cuda.synchronize()
        er, eg = lm.token_logprobs_and_grad(x, t, gl, top=3, entropy=True)
        for a, b in zip(res, er):
            assert torch.equal(a, b)
        assert torch.equal(g, eg)


def test_no_rows():
    x = torch.empty(0, 10, device="cuda")
    res, g = lm.token_logprobs_and_grad(x, torch.empty(0, dtype=torch.int64, device="cuda"),
                                        torch.empty(0, device="cuda"), top=2)
    assert res.logp.shape == (0,) and res.top_ids.shape == (0, 2) and g.shape == (0, 10)


def test_autograd_matches_differences():
    x, t = make(5, 40, torch.float32, std=1.0)
    t[2] = -100
    leaf = x.clone().requires_grad_()
    w = torch.linspace(0.5, 1.5, 5, device="cuda")
    logp, ent = lm.token_logp(leaf, t)
    ((logp + 0.3 * ent) * w).sum().backward()

    def loss(xd):
        r = ref.logprobs(xd, t)
        return ((r["logp"] + 0.3 * r["ent"]) * ref.d(w)).sum().item()

    v = torch.randn(5, 40, generator=torch.Generator().manual_seed(1), dtype=torch.float64)
    diff = (loss(ref.d(x) + 1e-4 * v) - loss(ref.d(x) - 1e-4 * v)) / 2e-4
    # central differences: third derivatives of order one times h^2 = 1e-8; float32 gradients
    assert abs((ref.d(leaf.grad) * v).sum().item() - diff) <= 1e-5 * 200


def test_evaluate_counts():
    x, t = make(50, 30, torch.bfloat16)
    t[:20] = x[:20].float().argmax(1)
    t[3] = -100
    loss, right, kept = lm.evaluate(x, t)
    want = ref.logprobs(x, t)
    assert int(kept) == 49 and int(right) == int(((best(x, 1)[:, 0] == t.cpu()) & (t.cpu() != -100)).sum())
    assert abs(float(loss) + float(want["logp"].sum())) <= 1e-3


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("R,V", [(767, 2049), (768, 2049), (769, 4099), (770, 16385)])
def test_many_rows(R, V, dtype):
    """Rows that fill the card, around the counts and lengths where a row's waves
    change; the alternatives are those of the pass without a gradient."""
    x, t = make(R, V, DT[dtype], seed=R)
    check(x, t, 0, DT[dtype], seed=1)
    a = lm.token_logprobs(x, t, top=3)
    b, _ = lm.token_logprobs_and_grad(x, t, torch.ones(R, device="cuda"), top=3)
    assert torch.equal(a.top_ids, b.top_ids)
    assert torch.equal(x.gather(1, a.top_ids[:, :1]).squeeze(1), x.max(1).values)

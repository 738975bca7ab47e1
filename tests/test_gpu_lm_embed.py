"""Embedding lookup with scaling and its gradient by sorted tokens (sra.h k13)."""
from __future__ import annotations

import math

import pytest
import torch

import lm_reference as ref
import srfl_amd.engine as engine
import srfl_amd.lm as lm

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def ids_of(T, V, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.exp(torch.rand(T, generator=g, dtype=torch.float64) * math.log(V + 1)) - 1).long().clamp(0, V - 1)


def rand(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def seg(offsets, slots):
    return torch.tensor(offsets, dtype=torch.int64).cuda(), torch.tensor(slots, dtype=torch.int32).cuda()


@pytest.mark.parametrize("tdtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("odtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("T,V,E", [(1, 1, 1), (5, 7, 3), (64, 50, 64), (33, 1000, 301), (3, 10, 4096)])
def test_lookup(T, V, E, tdtype, odtype):
    table, ids = rand(V, E, dtype=DT[tdtype]), ids_of(T, V).cuda()
    out = lm.embed(table, ids, scale=1.7, dtype=DT[odtype])
    assert torch.equal(out, (table.float()[ids] * 1.7).to(DT[odtype]))     # one float32 product, rounded once


def test_lookup_in_clients_tables_and_strided_rows():
    n, V, E = 4, 9, 10
    bank = rand(n, V * E + 5)
    table = bank[:, 3:3 + V * E].view(n, V, E)
    offsets, slots = [2, 6, 6, 11, 14], [3, 0, 1, -1]
    o, s = seg(offsets, slots)
    ids = ids_of(16, V).cuda()
    wide = torch.full((16, E + 4), 7.0, dtype=torch.bfloat16, device="cuda")
    lm.embed(table, ids, o, s, scale=2.0, out=wide[:, :E])
    slot = ref.token_slots(offsets, slots, 16).cuda()
    want = torch.where((slot >= 0)[:, None], table[slot.clamp(min=0), ids] * 2.0, 0.0).bfloat16()
    assert torch.equal(wide[:, :E], want) and (wide[:, E:] == 7).all()


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("T,V,E", [(1, 1, 1), (1, 5, 33), (7, 3, 8), (100, 40, 64), (33, 500, 301), (1000, 17, 20),
                                   (4095, 300, 12), (4096, 300, 12), (4097, 300, 12), (9001, 5000, 5), (65, 4, 2048)])
def test_gradient(T, V, E, dtype):
    dy, ids = rand(T, E, dtype=DT[dtype]), ids_of(T, V).cuda()
    grad = torch.full((V, E), 7.0, device="cuda")
    lm.embed_grad(dy, ids, grad, scale=1.5)
    want, bound = ref.embed_grad(dy, ids, 1, V, None, None, 1.5)
    ref.within("grad", grad, want[0], bound[0])
    untouched = torch.ones(V, dtype=torch.bool)
    untouched[ids.cpu()] = False
    assert not grad.cpu()[untouched].any()


@pytest.mark.parametrize("pattern", ["one_token", "two_tokens", "all_different", "descending"])
def test_gradient_runs(pattern):
    T, V, E = 5000, 6000, 24
    ids = {"one_token": torch.full((T,), 4321), "two_tokens": torch.arange(T) % 2 * 5999,
           "all_different": torch.randperm(V, generator=torch.Generator().manual_seed(1))[:T],
           "descending": V - 1 - torch.arange(T)}[pattern].cuda()
    dy = rand(T, E, dtype=torch.bfloat16)
    grad = lm.embed_grad(dy, ids, torch.empty(V, E, device="cuda"))
    want, bound = ref.embed_grad(dy, ids, 1, V, None, None, 1.0)
    ref.within(pattern, grad, want[0], bound[0])


@pytest.mark.parametrize("accumulate", [False, True])
def test_gradient_into_the_clients_matrix(accumulate):
    """Views of (n, D) rows, two segments of one client, gaps, padding, both modes."""
    n, V, E, T = 5, 21, 13, 300
    offsets, slots = [4, 80, 80, 150, 170, 280], [3, 1, 0, -1, 3]
    o, s = seg(offsets, slots)
    ids = ids_of(T, V).cuda()
    dy = rand(T, E, dtype=torch.bfloat16)
    dy[170:180] = 3.0
    G = torch.full((n, V * E + 3), 5.0, device="cuda")
    grad = G[:, 2:2 + V * E].view(n, V, E)
    lm.embed_grad(dy, ids, grad, o, s, scale=0.5, padding_idx=0, accumulate=accumulate)
    want, bound = ref.embed_grad(dy, ids, n, V, offsets, slots, 0.5, padding=0)
    if accumulate:
        want, bound = want + 5.0, bound + 2 * ref.U * (want.abs() + 5.0)
    ref.within("grad", grad, want, bound)
    assert (G[:, :2] == 5).all() and (G[:, -1] == 5).all()
    if accumulate:
        slot = ref.token_slots(offsets, slots, T)
        hit = torch.zeros(n, V, dtype=torch.bool)
        hit[slot[slot >= 0], ids.cpu()[slot >= 0]] = True
        hit[:, 0] = False
        assert (grad.cpu()[~hit] == 5.0).all()


def test_nan_in_rows_without_a_slot_stays_out():
    offsets, slots = [5, 40, 50], [1, -1]
    o, s = seg(offsets, slots)
    dy, ids = rand(64, 16, dtype=torch.bfloat16), ids_of(64, 9).cuda()
    a = lm.embed_grad(dy, ids, torch.empty(2, 9, 16, device="cuda"), o, s)
    dy[:5], dy[40:50], dy[50:] = float("nan"), float("inf"), float("nan")
    b = lm.embed_grad(dy, ids, torch.empty(2, 9, 16, device="cuda"), o, s)
    assert torch.equal(a, b) and torch.isfinite(a).all()


def test_repeats_bit_for_bit():
    dy, ids = rand(20000, 40, dtype=torch.bfloat16), ids_of(20000, 700).cuda()
    first = lm.embed_grad(dy, ids, torch.empty(700, 40, device="cuda"))
    for _ in range(3):
        assert torch.equal(first, lm.embed_grad(dy, ids, torch.empty(700, 40, device="cuda")))


def test_graph_replays():
    T, V, E = 5000, 120, 32
    table, ids, dy = rand(V, E), ids_of(T, V).cuda(), rand(T, E, dtype=torch.bfloat16)
    grad = torch.empty(V, E, device="cuda")
    graph = torch.cuda.CUDAGraph()
    lm.embed_grad(dy, ids, grad)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = lm.embed(table, ids, scale=3.0, dtype=torch.bfloat16)
        lm.embed_grad(dy, ids, grad)
    for i in range(4):
        ids.copy_(ids_of(T, V, seed=i))
        dy.copy_(rand(T, E, dtype=torch.bfloat16, seed=i))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, lm.embed(table, ids, scale=3.0, dtype=torch.bfloat16))
        assert torch.equal(grad, lm.embed_grad(dy, ids, torch.empty(V, E, device="cuda")))


def test_no_tokens():
    table = rand(3, 4)
    ids = torch.empty(0, dtype=torch.int64, device="cuda")
    assert lm.embed(table, ids).shape == (0, 4)
    grad = torch.full((3, 4), 5.0, device="cuda")
    lm.embed_grad(torch.empty(0, 4, device="cuda"), ids, grad, accumulate=True)
    assert (grad == 5).all()
    lm.embed_grad(torch.empty(0, 4, device="cuda"), ids, grad)
    assert not grad.any()


def test_bad_ids_are_counted():
    table, dy = rand(6, 8), rand(4, 8)
    ids = torch.tensor([1, 6, -1, 5]).cuda()
    engine.row_fault_count(reset=True)
    out = lm.embed(table, ids)
    assert engine.row_fault_count(reset=True) == 2
    assert torch.equal(out[[0, 3]], table[[1, 5]]) and not out[1:3].any()
    grad = lm.embed_grad(dy, ids, torch.empty(6, 8, device="cuda"))
    assert engine.row_fault_count(reset=True) == 2
    assert torch.equal(grad[1], dy[0]) and torch.equal(grad[5], dy[3]) and not grad[[0, 2, 3, 4]].any()


def test_autograd():
    table, ids, dy = rand(11, 6).requires_grad_(), ids_of(40, 11).cuda(), rand(40, 6, dtype=torch.bfloat16)
    (lm.embedding(table, ids, scale=2.0, dtype=torch.bfloat16) * dy).sum().backward()
    want, bound = ref.embed_grad(dy, ids, 1, 11, None, None, 2.0)
    ref.within("table.grad", table.grad, want[0], bound[0])


@pytest.mark.parametrize("T", [20000, 65536, 65537, 150001])
def test_gradient_of_more_tokens_than_one_merge_takes(T):
    """Runs of 4096 sorted tokens meet 16 at a time."""
    V, E = 700, 9
    dy, ids = rand(T, E, dtype=torch.bfloat16), ids_of(T, V)
    ids[::3] = torch.randint(0, V, ((T + 2) // 3,), generator=torch.Generator().manual_seed(3))
    ids = ids.cuda()
    offsets, slots = [1, T // 4, T // 2, T - 2], [1, 0, 1]
    o, s = seg(offsets, slots)
    grad = torch.full((2, V, E), 7.0, device="cuda")
    lm.embed_grad(dy, ids, grad, o, s, scale=0.5, padding_idx=3)
    want, bound = ref.embed_grad(dy, ids, 2, V, offsets, slots, 0.5, padding=3)
    ref.within("grad", grad, want, bound)
    # whole numbers add up without rounding: every token is in its row once
    ones = torch.ones(T, E, dtype=torch.bfloat16, device="cuda")
    lm.embed_grad(ones, ids, grad, o, s, padding_idx=3)
    want, _ = ref.embed_grad(ones, ids, 2, V, offsets, slots, 1.0, padding=3)
    assert torch.equal(grad.cpu().double(), want)


def test_many_segments():
    T, V, E, n = 3000, 40, 16, 6
    g = torch.Generator().manual_seed(2)
    offsets = torch.randint(0, T + 1, (901,), generator=g).sort().values.tolist()
    slots = torch.randint(-1, n, (900,), generator=g).tolist()
    o, s = seg(offsets, slots)
    table, ids, dy = rand(n, V, E), ids_of(T, V).cuda(), rand(T, E, dtype=torch.float16)
    slot = ref.token_slots(offsets, slots, T).cuda()
    want = torch.where((slot >= 0)[:, None], table[slot.clamp(min=0), ids] * 0.25, 0.0)
    assert torch.equal(lm.embed(table, ids, o, s, scale=0.25), want)
    grad = lm.embed_grad(dy, ids, torch.empty(n, V, E, device="cuda"), o, s)
    ref.within("grad", grad, *ref.embed_grad(dy, ids, n, V, offsets, slots, 1.0))

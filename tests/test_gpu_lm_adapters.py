"""Low-rank adapters of many clients beside a shared projection (sra.h k12)
against the formula in 64 bits (tests/lm_reference.py holds the bounds)."""
from __future__ import annotations

import pytest
import torch

import lm_reference as ref
import srfl_amd.engine as engine
import srfl_amd.lm as lm

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def make(T, K, M, r, n, dtype, wdtype, seed=0, pad_rows=0, pad_bank=0):
    g = torch.Generator().manual_seed(seed)

    def t(*shape, std=1.0):
        return torch.randn(*shape, generator=g) * std

    x = t(T, K + pad_rows).to(dtype).cuda()[:, :K]
    base = t(T, M + pad_rows).to(dtype).cuda()[:, :M]
    bank = (t(n, r * K + M * r + pad_bank) * 0.2).to(wdtype).cuda()
    A = bank[:, :r * K].view(n, r, K)
    B = bank[:, r * K:r * K + M * r].view(n, M, r)
    dy = t(T, M + pad_rows).to(dtype).cuda()[:, :M]
    dxb = t(T, K + pad_rows).to(dtype).cuda()[:, :K]
    return x, base, A, B, dy, dxb


def seg(offsets, slots):
    return torch.tensor(offsets, dtype=torch.int64).cuda(), torch.tensor(slots, dtype=torch.int32).cuda()


def check(T, K, M, r, n, offsets, slots, dtype, wdtype, scale=0.7, base=True, hidden=True, **kw):
    dtype, wdtype = DT[dtype], DT[wdtype]
    x, b, A, B, dy, dxb = make(T, K, M, r, n, dtype, wdtype, **kw)
    o, s = seg(offsets, slots)
    if not base:
        b = dxb = None
    want = ref.adapter(b, x, A, B, offsets, slots, scale, dtype, dy, dxb)
    y, h = lm.adapter_apply(b, x, A, B, o, s, scale, hidden=True)
    ref.within("out", y, *want["out"])
    dx, dA, dB = lm.adapter_grad(dy, x, A, B, o, s, scale, hidden=h if hidden else None, base_grad=dxb)
    ref.within("dx", dx, *want["dx"])
    ref.within("dA", dA, *want["dA"])
    ref.within("dB", dB, *want["dB"])
    assert y.dtype == dtype and dx.dtype == dtype and dA.dtype == dB.dtype == torch.float32
    return y, dx, dA, dB


@pytest.mark.parametrize("dtype,wdtype", [("bf16", "fp32"), ("bf16", "bf16"), ("fp16", "fp32"), ("fp16", "fp16"),
                                          ("fp32", "fp32")])
@pytest.mark.parametrize("T,K,M,r,offsets,slots", [
    (1, 1, 1, 1, [0, 1], [0]),
    (1, 64, 64, 8, [0, 1], [0]),
    (8, 128, 256, 8, list(range(9)), [7, 3, 1, 0, 2, 6, 5, 4]),
    (17, 100, 33, 5, [0, 16, 17], [1, 0]),
    (70, 129, 257, 16, [0, 1, 34, 70], [2, 0, 1]),
    (65, 320, 192, 17, [0, 65], [0]),
    (130, 96, 72, 33, [0, 63, 127, 130], [0, 1, 2]),
    (200, 520, 260, 64, [0, 150, 200], [1, 0]),
    (40, 1031, 7, 3, [0, 20, 40], [0, 1]),
])
def test_forward_and_gradients(T, K, M, r, offsets, slots, dtype, wdtype):
    check(T, K, M, r, max(8, max(slots) + 1), offsets, slots, dtype, wdtype)


@pytest.mark.parametrize("dtype,wdtype", [("bf16", "fp32"), ("fp32", "fp32")])
@pytest.mark.parametrize("case", ["empty_segments", "gaps", "none", "same_slot", "no_segment", "all_none"])
def test_segments(case, dtype, wdtype):
    T = 50
    offsets, slots = {
        "empty_segments": ([0, 0, 20, 20, 20, 50, 50], [0, 1, 2, 3, 0, 1]),
        "gaps": ([5, 21, 44], [1, 3]),                     # rows before the first and after the last segment
        "none": ([0, 10, 30, 50], [2, -1, 0]),
        "same_slot": ([0, 7, 25, 50], [1, 0, 1]),          # two segments of one client
        "no_segment": ([0], []),
        "all_none": ([0, 50], [-1]),
    }[case]
    y, dx, dA, dB = check(T, 72, 88, 8, 4, offsets, slots, dtype, wdtype)
    x, b, A, B, dy, dxb = make(T, 72, 88, 8, 4, DT[dtype], DT[wdtype])
    free = ref.token_slots(offsets, slots, T) < 0
    assert torch.equal(y.cpu()[free], b.cpu()[free]) and torch.equal(dx.cpu()[free], dxb.cpu()[free])
    for c in range(4):
        if c not in slots:
            assert not dA[c].any() and not dB[c].any()


@pytest.mark.parametrize("dtype,wdtype", [("bf16", "fp32"), ("bf16", "bf16"), ("fp16", "fp16"), ("fp32", "fp32")])
def test_strides_and_odd_alignment(dtype, wdtype):
    """Rows of wider matrices, client rows of odd length, no base, hidden computed again."""
    check(37, 75, 61, 7, 3, [0, 20, 37], [2, 0], dtype, wdtype, pad_rows=3, pad_bank=1)
    check(37, 75, 61, 7, 3, [0, 20, 37], [2, 0], dtype, wdtype, pad_rows=5, pad_bank=5, base=False, hidden=False)


def test_one_stretch_longer_than_any_tile():
    check(700, 200, 136, 16, 2, [0, 650, 700], [1, 0], "bf16", "fp32")
    check(700, 72, 40, 16, 2, [0, 699, 700], [1, 0], "fp32", "fp32")


def test_many_small_segments():
    offs = list(range(0, 301, 3))
    check(300, 64, 96, 4, 100, offs, [(7 * i) % 100 for i in range(100)], "bf16", "fp32")


def test_wide_rows_split_over_workgroups():
    check(3, 9000, 8200, 16, 3, [0, 1, 2, 3], [2, 1, 0], "bf16", "fp32")
    check(2, 5001, 4097, 64, 3, [0, 2], [2], "bf16", "bf16")


def test_in_place_and_views():
    x, base, A, B, dy, dxb = make(33, 64, 96, 8, 2, torch.bfloat16, torch.float32)
    o, s = seg([0, 10, 30], [1, 0])
    want = lm.adapter_apply(base, x, A, B, o, s, 2.0)
    wide = torch.full((33, 100), 7.0, dtype=torch.bfloat16, device="cuda")
    buf = wide[:, 2:98]
    buf.copy_(base)
    got = lm.adapter_apply(buf, x, A, B, o, s, 2.0, out=buf)
    assert got.data_ptr() == buf.data_ptr() and torch.equal(buf, want)
    assert (wide[:, :2] == 7).all() and (wide[:, 98:] == 7).all()
    dx, _, _ = lm.adapter_grad(dy, x, A, B, o, s, 2.0, base_grad=dxb, grad_A=False, grad_B=False)
    acc = dxb.clone()
    _, dA, dB = lm.adapter_grad(dy, x, A, B, o, s, 2.0, base_grad=acc, grad_x=acc)
    assert torch.equal(acc, dx) and dA is not None and dB is not None
    none = lm.adapter_grad(dy, x, A, B, o, s, grad_x=False, grad_A=False, grad_B=False)
    assert none == (None, None, None)


def test_gradient_rows_of_the_clients_matrix():
    """dA and dB as views of one (n, D) matrix of odd length; other columns untouched."""
    x, base, A, B, dy, dxb = make(40, 50, 30, 6, 4, torch.bfloat16, torch.float32)
    offsets, slots = [0, 15, 40], [3, 1]
    o, s = seg(offsets, slots)
    D = 50 * 6 + 30 * 6 + 3
    G = torch.full((4, D), 5.0, device="cuda")
    gA, gB = G[:, 1:301].view(4, 6, 50), G[:, 301:481].view(4, 30, 6)
    lm.adapter_grad(dy, x, A, B, o, s, 0.5, grad_A=gA, grad_B=gB)
    want = ref.adapter(base, x, A, B, offsets, slots, 0.5, torch.bfloat16, dy, dxb)
    ref.within("dA", gA, *want["dA"])
    ref.within("dB", gB, *want["dB"])
    assert (G[:, 0] == 5).all() and (G[:, 481:] == 5).all()
    before = G.clone()
    lm.adapter_grad(dy, x, A, B, o, s, 0.5, grad_A=gA, grad_B=gB, accumulate=True)
    ref.within("dA twice", gA, 2 * want["dA"][0], 2 * want["dA"][1] + 2 * ref.U * want["dA"][0].abs())
    ref.within("dB twice", gB, 2 * want["dB"][0], 2 * want["dB"][1] + 2 * ref.U * want["dB"][0].abs())
    assert torch.equal(G[[0, 2]], before[[0, 2]])          # slots without a token keep their values


def test_nan_and_inf_stay_where_they_are():
    x, base, A, B, dy, dxb = make(64, 80, 48, 8, 4, torch.bfloat16, torch.float32)
    offsets, slots = [3, 20, 40, 60], [0, -1, 1]
    o, s = seg(offsets, slots)
    y0 = lm.adapter_apply(base, x, A, B, o, s)
    g0 = lm.adapter_grad(dy, x, A, B, o, s, base_grad=dxb)
    x, dy, A, B = x.clone(), dy.clone(), A.clone(), B.clone()
    for bad, rows in ((float("nan"), slice(0, 3)), (float("inf"), slice(20, 40)), (float("nan"), slice(60, 64))):
        x[rows] = bad
        dy[rows] = bad
    A[2:], B[2:] = float("nan"), float("inf")
    assert torch.equal(lm.adapter_apply(base, x, A, B, o, s), y0)
    g1 = lm.adapter_grad(dy, x, A, B, o, s, base_grad=dxb)
    for a, b in zip(g0, g1):
        assert torch.equal(a, b)
    x[5, 7] = float("nan")                                   # one token's NaN stays with the token
    y2 = lm.adapter_apply(base, x, A, B, o, s)
    assert torch.isnan(y2[5]).all()
    keep = torch.arange(64) != 5
    assert torch.equal(y2.cpu()[keep], y0.cpu()[keep])


def test_infinite_weight():
    """A float32 operand w enters the matrix units as hi + rest, so a product with an
    infinity is inf * hi + inf * rest: the rest may be 0 or of the other sign, and the
    sum is then NaN where the formula has an infinity.  No finite value may come out,
    and the other clients' tokens keep theirs."""
    x, base, A, B, _, _ = make(4, 64, 32, 4, 2, torch.bfloat16, torch.float32)
    A, B = A.abs().contiguous(), B.abs().contiguous() + 0.1
    x = x.abs() + 0.5
    o, s = seg([0, 2, 4], [0, 1])
    y0 = lm.adapter_apply(base, x, A, B, o, s)
    A[0, 1, 3] = float("inf")
    y = lm.adapter_apply(base, x, A, B, o, s)
    assert not torch.isfinite(y[:2]).any() and torch.equal(y[2:], y0[2:])


def test_repeats_bit_for_bit_and_other_streams():
    x, base, A, B, dy, dxb = make(300, 256, 192, 16, 5, torch.bfloat16, torch.float32)
    o, s = seg([0, 100, 250, 300], [4, 0, 4])
    y, h = lm.adapter_apply(base, x, A, B, o, s, hidden=True)
    g = lm.adapter_grad(dy, x, A, B, o, s, hidden=h, base_grad=dxb)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(side):
            y2, h2 = lm.adapter_apply(base, x, A, B, o, s, hidden=True)
            g2 = lm.adapter_grad(dy, x, A, B, o, s, hidden=h2, base_grad=dxb)
        side.synchronize()
        assert torch.equal(y, y2) and torch.equal(h, h2)
        for a, b in zip(g, g2):
            assert torch.equal(a, b)


def test_graph_replays_with_new_values():
    """Inputs, offsets and slots change between replays; eager work runs in between."""
    x, base, A, B, dy, dxb = make(96, 128, 160, 8, 4, torch.bfloat16, torch.float32)
    o, s = seg([0, 40, 96], [1, 2])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        lm.adapter_apply(base, x, A, B, o, s)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, h = lm.adapter_apply(base, x, A, B, o, s, hidden=True)
        g = lm.adapter_grad(dy, x, A, B, o, s, hidden=h, base_grad=dxb)
    for i, (offs, sl) in enumerate([([0, 40, 96], [1, 2]), ([0, 1, 80], [3, -1]), ([10, 10, 96], [0, 3]),
                                    ([0, 96, 96], [2, 2])]):
        n = make(96, 128, 160, 8, 4, torch.bfloat16, torch.float32, seed=i + 1)
        for dst, src in zip((x, base, A, B, dy, dxb), n):
            dst.copy_(src)
        o.copy_(torch.tensor(offs))
        s.copy_(torch.tensor(sl, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        ye, he = lm.adapter_apply(base, x, A, B, o, s, hidden=True)
        ge = lm.adapter_grad(dy, x, A, B, o, s, hidden=he, base_grad=dxb)
        assert torch.equal(y, ye)
        for a, b in zip(g, ge):
            assert torch.equal(a, b)


def test_no_tokens():
    x, base, A, B, dy, dxb = make(4, 16, 24, 2, 3, torch.float32, torch.float32)
    o, s = seg([0, 0], [1])
    y, h = lm.adapter_apply(base[:0], x[:0], A, B, o, s, hidden=True)
    assert y.shape == (0, 24) and h.shape == (0, 2)
    dx, dA, dB = lm.adapter_grad(dy[:0], x[:0], A, B, o, s)
    assert dx.shape == (0, 16) and not dA.any() and not dB.any()


def test_bad_slots_and_offsets_are_counted_or_clamped():
    x, base, A, B, dy, dxb = make(20, 32, 32, 4, 2, torch.bfloat16, torch.float32)
    o, s = seg([0, 10, 20], [0, 1])
    good = lm.adapter_apply(base, x, A, B, o, s)
    o2, s2 = seg([0, 10, 20], [0, 9])
    engine.row_fault_count(reset=True)
    y = lm.adapter_apply(base, x, A, B, o2, s2)
    assert engine.row_fault_count(reset=True) > 0
    assert torch.equal(y[:10], good[:10]) and torch.equal(y[10:], base[10:])
    _, dA, dB = lm.adapter_grad(dy, x, A, B, o2, s2)
    assert engine.row_fault_count(reset=True) > 0 and not dA[1].any() and not dB[1].any()
    o3, s3 = seg([-5, 10, 4000], [0, 1])
    assert torch.equal(lm.adapter_apply(base, x, A, B, o3, s3), good)
    g, g3 = lm.adapter_grad(dy, x, A, B, o, s), lm.adapter_grad(dy, x, A, B, o3, s3)
    for a, b in zip(g, g3):
        assert torch.equal(a, b)


def test_autograd_matches_the_formula_and_differences():
    x, base, A, B, dy, dxb = make(12, 20, 14, 3, 2, torch.float32, torch.float32)
    offsets, slots = [0, 5, 12], [1, 0]
    o, s = seg(offsets, slots)
    leaves = [t.clone().requires_grad_() for t in (base, x, A, B)]
    (lm.adapters(*leaves, o, s, 0.7) * dy).sum().backward()
    want = ref.adapter(base, x, A, B, offsets, slots, 0.7, torch.float32, dy, None)
    assert torch.equal(leaves[0].grad, dy)
    for leaf, name in zip(leaves[1:], ("dx", "dA", "dB")):
        ref.within(name, leaf.grad, *want[name])

    def loss(xd, Ad, Bd):
        r = ref.adapter(base, xd, Ad, Bd, offsets, slots, 0.7, torch.float32)
        return (r["out"][0] * ref.d(dy)).sum().item()

    g = torch.Generator().manual_seed(3)
    args = [ref.d(t) for t in (x, A, B)]
    for i, leaf in enumerate(leaves[1:]):
        v = torch.randn(args[i].shape, generator=g, dtype=torch.float64)
        lo, hi = list(args), list(args)
        lo[i], hi[i] = args[i] - 1e-4 * v, args[i] + 1e-4 * v
        diff = (loss(*hi) - loss(*lo)) / 2e-4              # the loss is quadratic at most in one argument
        assert abs((ref.d(leaf.grad) * v).sum().item() - diff) <= 1e-4 * max(1.0, abs(diff))


@pytest.mark.parametrize("T,count,step,dtype,wdtype", [
    (300, 255, 1, "bf16", "fp32"), (300, 256, 1, "fp32", "fp32"), (9000, 5000, 1, "bf16", "fp32"),
    (9000, 257, 35, "bf16", "bf16"), (9000, 258, 34, "fp32", "fp32"),
])
def test_more_segments_than_one_round_of_loads(T, count, step, dtype, wdtype):
    """Segments of `step` tokens with empty ones and rows of no segment between them."""
    g = torch.Generator().manual_seed(count)
    sizes = step * torch.ones(count, dtype=torch.int64)
    sizes[torch.randperm(count, generator=g)[:count // 5]] = 0
    offsets = [2] + (2 + sizes.cumsum(0)).clamp(max=T).tolist()
    slots = torch.randint(-1, 5, (count,), generator=g).tolist()
    check(T, 24, 16, 3, 5, offsets, slots, dtype, wdtype)


@pytest.mark.parametrize("T,K,M,r,n,dtype", [
    (2000, 75, 64, 16, 1, "bf16"),        # few columns in all: waves share columns, parts of the tokens
    (1500, 33, 300, 40, 2, "fp32"),
    (700, 515, 8, 4, 100, "bf16"),        # a wave its own columns, the last ones of a row not whole
    (33000, 513, 24, 8, 100, "fp16"),     # the same, parts of the tokens
])
def test_gradient_sums_split_over_workgroups(T, K, M, r, n, dtype):
    slots = [n - 1, 0, 1 % n] + list(range(2, n - 1))          # the last ones are empty
    offsets = [0, T // 3, T // 3 + 1, T - 5] + [T - 5] * (len(slots) - 3)
    x, base, A, B, dy, dxb = make(T, K, M, r, n, DT[dtype], torch.float32)
    o, s = seg(offsets, slots)
    want = ref.adapter(base, x, A, B, offsets, slots, 0.5, DT[dtype], dy, dxb)
    _, gA, gB = lm.adapter_grad(dy, x, A, B, o, s, 0.5)
    ref.within("dA", gA, *want["dA"])
    ref.within("dB", gB, *want["dB"])
    gA, gB = torch.full_like(gA, 5.0), torch.full_like(gB, 5.0)
    lm.adapter_grad(dy, x, A, B, o, s, 0.5, grad_A=gA, grad_B=gB, accumulate=True)
    for name, got, (val, err) in (("dA", gA, want["dA"]), ("dB", gB, want["dB"])):
        ref.within(name + " added", got, val + 5.0, err + 2 * ref.U * (val.abs() + 5.0))
    for c in range(n):
        if all(q != c or offsets[i] == offsets[i + 1] for i, q in enumerate(slots)):
            assert (gA[c] == 5.0).all() and (gB[c] == 5.0).all()


def test_rows_far_apart():
    """Row strides that put offsets beyond 2^31 elements."""
    T, K, M = 20, 40, 24
    ld = (1 << 31) // 16
    x, base, A, B, dy, dxb = make(T, K, M, 4, 2, torch.bfloat16, torch.float32)
    o, s = seg([0, 7, 20], [1, 0])
    far = torch.empty(T * ld, dtype=torch.bfloat16, device="cuda").view(T, ld)
    fx, fb, fy, fo, fd = (far[:, i * 64:][:, :w] for i, w in enumerate((K, M, M, M, K)))
    fx.copy_(x), fb.copy_(base), fy.copy_(dy)
    y = lm.adapter_apply(base, x, A, B, o, s)
    lm.adapter_apply(fb, fx, A, B, o, s, out=fo)
    assert torch.equal(fo, y)
    near = lm.adapter_grad(dy, x, A, B, o, s)
    dx, gA, gB = lm.adapter_grad(fy, fx, A, B, o, s, grad_x=fd)
    assert torch.equal(fd, near[0]) and torch.equal(gA, near[1]) and torch.equal(gB, near[2])


def test_two_graphs_and_eager_calls_in_turn():
    """Each graph has workspaces of its own."""
    cases = []
    for i, (T, n) in enumerate([(300, 3), (2100, 1)]):
        x, base, A, B, dy, dxb = make(T, 640, 520, 8, n, torch.bfloat16, torch.float32, seed=i)
        o, s = seg([0, T // 2, T], [n - 1, 0])
        lm.adapter_apply(base, x, A, B, o, s)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y, h = lm.adapter_apply(base, x, A, B, o, s, hidden=True)
            got = (y,) + lm.adapter_grad(dy, x, A, B, o, s, hidden=h, base_grad=dxb)
        cases.append((graph, got, (x, base, A, B, dy, dxb, o, s)))
    for _ in range(3):
        for graph, got, _ in cases:
            for t in got:
                t.fill_(float("nan"))
            graph.replay()
        for _, got, (x, base, A, B, dy, dxb, o, s) in cases:
            y, h = lm.adapter_apply(base, x, A, B, o, s, hidden=True)
            for a, b in zip(got, (y,) + lm.adapter_grad(dy, x, A, B, o, s, hidden=h, base_grad=dxb)):
                assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T,K,M,r,offsets,slots", [
    (70, 129, 257, 16, [0, 1, 34, 70], [2, 0, 1]), (200, 520, 260, 64, [0, 150, 200], [1, 0]),
    (20, 300, 90, 24, list(range(21)), [i % 3 for i in range(20)]),
])
def test_float32_weights_and_gradients_keep_their_bits(T, K, M, r, offsets, slots, dtype, monkeypatch):
    """Hidden values and gradients stay float32: three bf16 terms hold a float32's
    24 bits, two an fp16's 11, and what is left out of their products is below
    2^-8 * 2^-16 of one, twice: 2^-22 bounds it beside the float32 sums."""
    monkeypatch.setattr(ref, "PROD", 2.0 ** -22)
    x, base, A, B, dy, dxb = make(T, K, M, r, 3, DT[dtype], torch.float32)
    o, s = seg(offsets, slots)
    want = ref.adapter(base, x, A, B, offsets, slots, 0.7, DT[dtype], dy, dxb)
    _, h = lm.adapter_apply(base, x, A, B, o, s, 0.7, hidden=True)
    _, dA, dB = lm.adapter_grad(dy, x, A, B, o, s, 0.7, hidden=h)
    ref.within("dA", dA, *want["dA"])
    ref.within("dB", dB, *want["dB"])
    for a, b, c in ref.segments(offsets, slots, T):
        v, e = ref.product(ref.d(x[a:b]), torch.zeros(b - a, K).double(), ref.d(A[c]).T.contiguous(),
                           torch.zeros(K, r).double())
        ref.within("hidden", h[a:b], v, e)


@pytest.mark.parametrize("T,K,M,r,dtype,wdtype", [
    (700, 1001, 777, 5, "fp32", "fp32"), (300, 1024, 1500, 16, "bf16", "bf16"), (300, 1040, 2050, 16, "fp16", "fp32"),
    (130, 4100, 520, 33, "bf16", "fp32"), (64, 9000, 300, 1, "bf16", "bf16"),
])
def test_few_tiles_share_the_width(T, K, M, r, dtype, wdtype):
    """Hidden values as partial sums of the width, some parts of them empty."""
    check(T, K, M, r, 2, [0, T // 2 + 3, T], [1, 0], dtype, wdtype)
    check(T, K, M, r, 2, [0, T // 2 + 3, T], [1, 0], dtype, wdtype, base=False, hidden=False, pad_rows=1)

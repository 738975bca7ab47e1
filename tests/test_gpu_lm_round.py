"""The language-model operators together, as one federated round uses them:
every client's embedding and adapters train at once on rows of a ClientBank,
fl_round aggregates and applies, evaluate gives the results row."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import lm_reference as ref
from srfl_amd import dispatch, formats, lm, store

pytestmark = pytest.mark.gpu

V, E, H, R = 37, 24, 40, 4          # vocabulary, embedding, hidden, adapter rank
SHAPES = [(V, E), (R, E), (H, R)]   # what a client trains: embedding, A, B


class Net:
    """A shared projection and output layer that stay fixed beside what the clients train."""

    def __init__(self, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.params = [(0.3 * torch.randn(s, generator=g)).cuda() for s in SHAPES]
        self.W = (torch.randn(H, E, generator=g) / E ** 0.5).cuda()
        self.O = (torch.randn(V, H, generator=g) / H ** 0.5).cuda()

    def parameters(self):
        return self.params


def batch(n, seed=0):
    g = torch.Generator().manual_seed(seed)
    lens = torch.randint(1, 30, (n,), generator=g)
    lens[0] = 1
    offsets = [0] + torch.cumsum(lens, 0).tolist()
    T = offsets[-1]
    ids = torch.randint(0, V, (T,), generator=g)
    targets = (ids * 5 + 3) % V
    targets[::7] = -100
    return offsets, ids, targets


def loss_and_grads(net, tables, A, B, offsets, slots, ids, targets, scale, w):
    """Plain float64 autograd: gradients of every client's embedding and adapter."""
    t, a, b = [ref.d(p).requires_grad_() for p in (tables, A, B)]
    W, O = ref.d(net.W), ref.d(net.O)
    total = 0.0
    for lo, hi, c in ref.segments(offsets, slots, len(ids)):
        x = t[c][ids[lo:hi]] * 2.0
        y = x @ W.T + scale * (x @ a[c].T) @ b[c].T
        lp = torch.log_softmax(y @ O.T, dim=1)
        keep = targets[lo:hi] >= 0
        total = total + (lp.gather(1, targets[lo:hi].clamp(min=0)[:, None]).squeeze(1) * w[lo:hi])[keep].sum()
    total.backward()
    return t.grad, a.grad, b.grad


def train_step(net, bank, offsets, slots, ids, targets, w, scale=0.5):
    """One local step of all clients with the explicit operators."""
    tables, A, B = bank.param(0), bank.param(1), bank.param(2)
    x = lm.embed(tables, ids, offsets, slots, scale=2.0)
    y, hidden = lm.adapter_apply(x @ net.W.T, x, A, B, offsets, slots, scale, hidden=True)
    logits = y @ net.O.T
    res, dlogits = lm.token_logprobs_and_grad(logits, targets, w, out=logits)
    dy = dlogits @ net.O
    dx, _, _ = lm.adapter_grad(dy, x, A, B, offsets, slots, scale, hidden, base_grad=dy @ net.W,
                               grad_A=bank.grad(1), grad_B=bank.grad(2))
    lm.embed_grad(dx, ids, bank.grad(0), offsets, slots, scale=2.0)
    return res


def test_gradients_of_all_clients_land_in_their_rows():
    n = 6
    net = Net()
    S = store.ClientStore(net.parameters(), n)
    S.snapshot()
    bank = store.ClientBank(S, n)
    bank.load(range(n))
    bank.P.add_(0.1 * torch.randn(bank.P.shape, generator=torch.Generator().manual_seed(1)).cuda())
    offsets, ids, targets = batch(n)
    slots = [3, 0, 5, 1, 4, 2]
    T = len(ids)
    w = torch.full((T,), -1.0 / T)
    o, s = torch.tensor(offsets).cuda(), torch.tensor(slots, dtype=torch.int32).cuda()
    train_step(net, bank, o, s, ids.cuda(), targets.cuda(), w.cuda())
    want = loss_and_grads(net, bank.param(0), bank.param(1), bank.param(2), offsets, slots, ids, targets, 0.5, ref.d(w))
    for l in range(3):
        got = ref.d(bank.grad(l))
        # five float32 products of at most 40 terms each, and PROD of the adapters': relative to the largest gradient
        assert (got - want[l]).abs().max() <= 5 * (40 * ref.U + ref.PROD) * 8 * want[l].abs().max()


def test_autograd_forms_give_the_same_gradients():
    n = 5
    net = Net(2)
    S = store.ClientStore(net.parameters(), n)
    S.snapshot()
    bank = store.ClientBank(S, n)
    bank.load(range(n))
    offsets, ids, targets = batch(n, 3)
    slots = list(range(n))
    T = len(ids)
    w = torch.full((T,), -1.0 / T).cuda()
    o, s = torch.tensor(offsets).cuda(), torch.tensor(slots, dtype=torch.int32).cuda()
    train_step(net, bank, o, s, ids.cuda(), targets.cuda(), w)
    leaves = [bank.param(l).detach().clone().requires_grad_() for l in range(3)]
    x = lm.embedding(leaves[0], ids.cuda(), o, s, scale=2.0)
    y = lm.adapters(x @ net.W.T, x, leaves[1], leaves[2], o, s, 0.5)
    logp, _ = lm.token_logp(y @ net.O.T, targets.cuda())
    (logp * w).sum().backward()
    for l in range(3):
        got, want = ref.d(leaves[l].grad), ref.d(bank.grad(l))
        assert (got - want).abs().max() <= 10 * (40 * ref.U + ref.PROD) * 8 * want.abs().max()


@pytest.mark.parametrize("agg", ["average", "trimmedmean", "krum", "iclr2022_bucketing"])
def test_round_matches_clients_one_after_another(agg, tmp_path):
    """fl_round with a bank against fl_round with the clients in turn, which use the
    same operators with one client's rows: the store's updates and the applied
    parameters are the same."""
    n = 12
    momentum = agg == "iclr2022_bucketing"
    offsets, ids, targets = batch(n, 5)
    choices = np.random.RandomState(0).permutation(n)
    args = dispatch.RoundArgs(agg=agg, nworker=n, perround=n, malnum=2, buckets=3)
    T = len(ids)

    def at_once(net, S):
        bank = store.ClientBank(S, n)
        o = torch.tensor(offsets).cuda()
        s = torch.arange(n, dtype=torch.int32).cuda()

        def train(bk):
            for _ in range(2):
                train_step(net, bk, o, s, ids.cuda(), targets.cuda(), torch.full((T,), -0.05).cuda())
                bk.step(0.5)
        return dict(local_update=train, bank=bank)

    def in_turn(net, S):
        def train(c):
            i = int(np.nonzero(choices == c)[0][0])
            lo, hi = offsets[i], offsets[i + 1]
            o = torch.tensor([0, hi - lo]).cuda()
            s = torch.zeros(1, dtype=torch.int32).cuda()

            class One:
                def param(self, l):
                    return net.params[l][None]

                def grad(self, l):
                    return grads[l][None]
            grads = [torch.empty_like(p) for p in net.params]
            for _ in range(2):
                train_step(net, One(), o, s, ids[lo:hi].cuda(), targets[lo:hi].cuda(),
                           torch.full((hi - lo,), -0.05).cuda())
                for p, g in zip(net.params, grads):
                    p.add_(g, alpha=-0.5)
        return dict(local_update=train)

    flats, nets, updates = [], [], []
    for how in (at_once, in_turn):
        net = Net(4)
        S = store.ClientStore(net.parameters(), n, momentum=momentum)
        np.random.seed(1)
        kw = how(net, S)
        ch = choices.copy()
        flats.append(store.fl_round(net, S, ch, kw["local_update"], args, dispatch.DispatchState(),
                                    bank=kw.get("bank")))
        nets.append(net)
        updates.append(S.U.clone())
    # the two differ by the order of float32 sums only (library products of other shapes among them)
    top = updates[1].abs().max().item()
    assert (updates[0] - updates[1]).abs().max().item() <= 2 * 5 * (40 * ref.U + ref.PROD) * 8 * top
    if agg != "krum":               # krum may take another client on a near-tie
        assert (flats[0].double() - flats[1].double()).abs().max().item() <= 10 * (40 * ref.U + ref.PROD) * 8 * top
    net = nets[0]
    x = lm.embed(net.params[0], ids.cuda(), scale=2.0)
    o, s = torch.tensor([0, T]).cuda(), torch.zeros(1, dtype=torch.int32).cuda()
    y = lm.adapter_apply(x @ net.W.T, x, net.params[1][None], net.params[2][None], o, s, 0.5)
    loss, right, kept = lm.evaluate(y @ net.O.T, targets.cuda())
    row = formats.format_result_row(1, loss / kept, 100.0 * right / kept)
    assert np.isfinite(formats.parse_results(row + "\n")).all()


def test_bank_refuses_other_clients():
    net = Net()
    S = store.ClientStore(net.parameters(), 4)
    S.snapshot()
    with pytest.raises(ValueError, match="bank"):
        store.ClientBank(S, 5)
    bank = store.ClientBank(S, 2)
    with pytest.raises(RuntimeError, match="choices"):
        bank.record()
    with pytest.raises(ValueError, match="different"):
        bank.load([1, 1])
    with pytest.raises(ValueError, match="different"):
        bank.load([0, 1, 2])
    with pytest.raises(IndexError):
        bank.load([0, 4])


def test_autograd_forms_refuse_capture():
    net = Net()
    ids = torch.arange(5).cuda()
    table = net.params[0].clone().requires_grad_()
    lm.embedding(table, ids)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(graph):
            lm.embedding(table, ids)
    with torch.no_grad():
        assert lm.embedding(table, ids).shape == (5, E)


def test_round_refuses_a_bank_of_another_store():
    net = Net()
    S, other = (store.ClientStore(net.parameters(), 4) for _ in range(2))
    before = [p.clone() for p in net.params]
    with pytest.raises(ValueError, match="another store"):
        store.fl_round(net, S, [0, 1], lambda bank: bank.step(1.0), None, bank=store.ClientBank(other, 2))
    assert all(torch.equal(p, q) for p, q in zip(net.params, before))

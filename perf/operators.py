"""Measured cases of the language-model client operators (``srfl_amd.lm``).

Three operators that a federated round over language-model clients runs next to
the client-major (N, D) matrix of the aggregators:

* ``adapters`` -- every client's low-rank adapter beside a shared projection,
  ``y_t = base_t + scale * B_c (A_c x_t)`` for the tokens t of client c, and the
  gradients of x, A and B;
* ``embed``    -- embedding lookup with scaling from one shared table or one
  table a client, and the table's gradient summed token by token;
* ``logprobs`` -- log probabilities of given tokens with the entropy and the
  top alternatives of every row, alone or with the gradient of the logits.

The adapters and the tables a client trains are float32 (rows of the clients'
matrix); activations and logits are bfloat16, float16 or float32.  Client
counts follow the framework's own workloads (100 and 128 clients).
"""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # one decoding step of a few requests, each with an adapter of its own, served in bf16
        dict(name="adapters_step_small", op="adapters", train=False, tokens=8, segments=8, clients=8, k=1024, m=1024,
             rank=8, dtype="bf16", weights="bf16"),
        # one decoding step of 100 clients' candidate adapters, straight from the float32 client rows
        dict(name="adapters_step_100", op="adapters", train=False, tokens=100, segments=100, clients=100, k=4096,
             m=4096, rank=16, dtype="bf16", weights="fp32"),
        # evaluation of 32 clients' adapters on ragged prompts
        dict(name="adapters_eval", op="adapters", train=False, tokens=8192, segments=32, clients=32, k=4096, m=4096,
             rank=16, dtype="bf16", weights="fp32"),
        # a local training step of 100 clients at once, ragged batches, gradients into the client rows
        dict(name="adapters_train_100", op="adapters", train=True, tokens=6400, segments=100, clients=100, k=2048,
             m=2048, rank=16, dtype="bf16", weights="fp32"),
        # a float32 training step with odd sizes throughout
        dict(name="adapters_train_odd", op="adapters", train=True, tokens=1501, segments=11, clients=13, k=1001,
             m=777, rank=5, dtype="fp32", weights="fp32"),
        # a long-context training step of 16 clients at a large rank
        dict(name="adapters_train_large", op="adapters", train=True, tokens=16384, segments=16, clients=16, k=8192,
             m=8192, rank=64, dtype="bf16", weights="fp32"),
        # lookup for one decoding step of 100 clients, each in its own table
        dict(name="embed_step", op="embed", train=False, tokens=100, segments=100, clients=100, vocab=4001, dim=1024,
             dtype="bf16"),
        # training on one shared table: lookup and gradient, tokens of a skewed distribution
        dict(name="embed_train_shared", op="embed", train=True, tokens=32768, segments=0, clients=1, vocab=50001,
             dim=2048, dtype="bf16"),
        # training of 100 clients' own tables on ragged batches: gradients into the client rows
        dict(name="embed_train_clients", op="embed", train=True, tokens=25600, segments=100, clients=100, vocab=8192,
             dim=300, dtype="fp32"),
        # sampling step: a few rows, five alternatives
        dict(name="logprobs_step", op="logprobs", train=False, rows=8, vocab=32768, top=5, dtype="bf16"),
        # evaluation of given tokens over a large vocabulary: loss, entropy and top-1 accuracy
        dict(name="logprobs_eval", op="logprobs", train=False, rows=4096, vocab=131072, top=1, dtype="bf16"),
        # the training loss over an odd vocabulary, some tokens ignored, with the logits' gradient
        dict(name="logprobs_train", op="logprobs", train=True, rows=4096, vocab=50001, top=0, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["adapters", "adapters", "embed", "logprobs"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    train = rng.random() < 0.5
    if op == "adapters":
        segments = _log_int(rng, 1, 128)
        k, m = _log_int(rng, 64, 8192), _log_int(rng, 64, 8192)
        if rng.random() < 0.6:      # widths of real layers are multiples of 64 more often than not
            k, m = -(-k // 64) * 64, -(-m // 64) * 64
        most = (1 << 28) // ((k + m) * _SIZE[dtype])
        return dict(op=op, train=train, tokens=max(segments, _log_int(rng, 1, min(16384, most))), segments=segments,
                    clients=segments + rng.randrange(0, 4), k=k, m=m, rank=_log_int(rng, 1, 64), dtype=dtype,
                    weights="fp32" if train or rng.random() < 0.5 else dtype)
    if op == "embed":
        clients = rng.choice([1, 1, _log_int(rng, 2, 128)])
        dim = _log_int(rng, 16, 4096)
        vocab = _log_int(rng, 100, max(101, min(131072, (1 << 28) // (clients * dim))))
        segments = 0 if clients == 1 else clients
        return dict(op=op, train=train, tokens=max(clients, _log_int(rng, 1, 32768)), segments=segments,
                    clients=clients, vocab=vocab, dim=dim, dtype=dtype)
    vocab = _log_int(rng, 10, 131072)
    rows = _log_int(rng, 1, max(1, min(8192, (1 << 27) // vocab)))
    return dict(op=op, train=train, rows=rows, vocab=vocab, top=0 if train else rng.randrange(0, min(vocab, 20) + 1),
                dtype=dtype)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _offsets(tokens, segments, seed):
    """Ragged segments that cover the tokens, one token each at least."""
    g = torch.Generator().manual_seed(int(seed) + 77)
    cuts = torch.randperm(tokens - 1, generator=g)[:segments - 1].sort().values + 1 if segments > 1 else []
    return [0] + [int(c) for c in cuts] + [tokens]


def _slots(segments, clients, seed):
    g = torch.Generator().manual_seed(int(seed) + 78)
    return [int(c) for c in torch.randperm(clients, generator=g)[:segments]]


def _ids(tokens, vocab, gen):
    """Token ids with a frequency that falls like one over the rank."""
    u = torch.rand(tokens, generator=gen, device="cuda", dtype=torch.float64)
    return (torch.exp(u * math.log(vocab + 1)) - 1).long().clamp_(0, vocab - 1)


def prepare(case, seed):
    g = _gen(seed)
    dt = _DT[case["dtype"]]

    def randn(*shape, dtype=dt, std=1.0):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).mul_(std).to(dtype)

    st = dict(case=case)
    if case["op"] == "adapters":
        T, K, M, r, n = case["tokens"], case["k"], case["m"], case["rank"], case["clients"]
        wdt = _DT[case["weights"]]
        st["host_offsets"] = _offsets(T, case["segments"], seed)
        st["host_slots"] = _slots(case["segments"], n, seed)
        st["offsets"] = torch.tensor(st["host_offsets"], dtype=torch.int64, device="cuda")
        st["slots"] = torch.tensor(st["host_slots"], dtype=torch.int32, device="cuda")
        st["scale"] = 2.0
        st["x"] = randn(T, K)
        st["base"] = randn(T, M)
        # a client's trainable parameters are one row of the clients' matrix: A then B
        st["bank"] = randn(n, r * K + M * r, dtype=wdt, std=1.0 / math.sqrt(K))
        st["A"] = st["bank"][:, :r * K].view(n, r, K)
        st["B"] = st["bank"][:, r * K:].view(n, M, r)
        if case["train"]:
            st["dy"] = randn(T, M, std=1.0 / math.sqrt(M))
            st["dx_base"] = randn(T, K)
            st["grads"] = torch.empty(n, r * K + M * r, dtype=torch.float32, device="cuda")
    elif case["op"] == "embed":
        T, V, E, n = case["tokens"], case["vocab"], case["dim"], case["clients"]
        st["ids"] = _ids(T, V, g)
        st["scale"] = math.sqrt(E)
        st["table"] = randn(n, V, E, dtype=torch.float32, std=0.02)
        st["host_offsets"] = _offsets(T, case["segments"], seed) if case["segments"] else [0, T]
        st["host_slots"] = _slots(case["segments"], n, seed) if case["segments"] else [0]
        if case["segments"]:
            st["offsets"] = torch.tensor(st["host_offsets"], dtype=torch.int64, device="cuda")
            st["slots"] = torch.tensor(st["host_slots"], dtype=torch.int32, device="cuda")
        else:
            st["offsets"] = st["slots"] = None
        if case["train"]:
            st["dy"] = randn(T, E)
            st["grad"] = torch.empty(n, V, E, dtype=torch.float32, device="cuda")
    else:
        T, V = case["rows"], case["vocab"]
        st["targets"] = _ids(T, V, g)
        x = torch.randn(T, V, generator=g, device="cuda", dtype=torch.float32).mul_(2.0)
        # a model that has learned something: the given token stands out in most rows
        lift = torch.rand(T, 1, generator=g, device="cuda") * 12.0
        x.scatter_add_(1, st["targets"].view(-1, 1), lift)
        st["logits"] = x.to(dt)
        del x
        if case["train"]:
            ignored = torch.rand(T, generator=g, device="cuda") < 0.1
            st["targets"] = torch.where(ignored, torch.full_like(st["targets"], -100), st["targets"])
            kept = max(1, int((~ignored).sum()))
            st["weights"] = torch.where(ignored, 0.0, -1.0 / kept).float()
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if own:
        return {"adapters": _own_adapters, "embed": _own_embed, "logprobs": _own_logprobs}[op](state)
    return {"adapters": _plain_adapters, "embed": _plain_embed, "logprobs": _plain_logprobs}[op](state)


_module = None


def _lm():
    global _module
    if _module is None:
        import srfl_loader
        srfl_loader.load()
        from srfl_amd import lm
        _module = lm
    return _module


def _own_adapters(st):
    lm = _lm()
    if not st["case"]["train"]:
        return lm.adapter_apply(st["base"], st["x"], st["A"], st["B"], st["offsets"], st["slots"], st["scale"])
    r, K, M = st["case"]["rank"], st["case"]["k"], st["case"]["m"]
    n = st["case"]["clients"]
    y, hidden = lm.adapter_apply(st["base"], st["x"], st["A"], st["B"], st["offsets"], st["slots"], st["scale"],
                                 hidden=True)
    dA = st["grads"][:, :r * K].view(n, r, K)
    dB = st["grads"][:, r * K:].view(n, M, r)
    # float32 training adds to dx_base where it lies, as the plain form does (its conversion is no copy there)
    in_place = st["dx_base"].dtype is torch.float32
    dx, _, _ = lm.adapter_grad(st["dy"], st["x"], st["A"], st["B"], st["offsets"], st["slots"], st["scale"],
                               hidden=hidden, base_grad=st["dx_base"], grad_x=st["dx_base"] if in_place else True,
                               grad_A=dA, grad_B=dB)
    return y, dx, st["grads"]


def _own_embed(st):
    lm = _lm()
    dt = _DT[st["case"]["dtype"]]
    table = st["table"] if st["offsets"] is not None else st["table"][0]
    out = lm.embed(table, st["ids"], st["offsets"], st["slots"], scale=st["scale"], dtype=dt)
    if not st["case"]["train"]:
        return out
    grad = st["grad"] if st["offsets"] is not None else st["grad"][0]
    lm.embed_grad(st["dy"], st["ids"], grad, st["offsets"], st["slots"], scale=st["scale"])
    return out, st["grad"]


def _own_logprobs(st):
    lm = _lm()
    if st["case"]["train"]:
        res, grad = lm.token_logprobs_and_grad(st["logits"], st["targets"], st["weights"])
        return res.logp, grad
    res = lm.token_logprobs(st["logits"], st["targets"], top=st["case"]["top"], entropy=True)
    if st["case"]["top"] == 0:
        return res.logp, res.entropy
    return res.logp, res.entropy, res.top_logp, res.top_ids


def _segments(st):
    o = st["host_offsets"]
    return [(o[s], o[s + 1], c) for s, c in enumerate(st["host_slots"])]


def _plain_adapters(st):
    scale, train = st["scale"], st["case"]["train"]
    x, base = st["x"].float(), st["base"].float()
    A, B = st["A"].float(), st["B"].float()
    y = base.clone()
    if train:
        dy = st["dy"].float()
        dx = st["dx_base"].float()
        st["grads"].zero_()
        r, K, M = st["case"]["rank"], st["case"]["k"], st["case"]["m"]
        n = st["case"]["clients"]
        dA = st["grads"][:, :r * K].view(n, r, K)
        dB = st["grads"][:, r * K:].view(n, M, r)
    for a, b, c in _segments(st):
        h = x[a:b] @ A[c].t()
        y[a:b] += scale * (h @ B[c].t())
        if train:
            z = dy[a:b] @ B[c]
            dx[a:b] += scale * (z @ A[c])
            dA[c] = scale * (z.t() @ x[a:b])
            dB[c] = scale * (dy[a:b].t() @ h)
    y = y.to(st["base"].dtype)
    return (y, dx.to(st["dx_base"].dtype), st["grads"]) if train else y


def _rows_of(st):
    """Row of the (clients * vocab, dim) table that every token reads."""
    o = torch.tensor(st["host_offsets"], device="cuda")
    lengths = o[1:] - o[:-1]
    slot = torch.tensor(st["host_slots"], device="cuda").repeat_interleave(lengths)
    return slot * st["case"]["vocab"] + st["ids"]


def _plain_embed(st):
    n, V, E = st["table"].shape
    rows = _rows_of(st)
    out = (st["table"].view(n * V, E)[rows] * st["scale"]).to(_DT[st["case"]["dtype"]])
    if not st["case"]["train"]:
        return out
    # every row's tokens summed in 64 bits, a block of columns at a time
    step = max(1, min(E, (1 << 28) // (n * V)))
    for e in range(0, E, step):
        acc = torch.zeros(n * V, min(step, E - e), dtype=torch.float64, device="cuda")
        acc.index_add_(0, rows, st["dy"][:, e:e + step].double())
        st["grad"].view(n * V, E)[:, e:e + step] = (acc * st["scale"]).float()
    return out, st["grad"]


def _plain_logprobs(st):
    x = st["logits"].float()
    t = st["targets"]
    V = x.shape[1]
    kept = t >= 0
    m = x.max(dim=1, keepdim=True).values
    e = torch.exp(x - m)
    s = e.sum(dim=1, keepdim=True)
    lse = m + torch.log(s)
    at = t.clamp(min=0).view(-1, 1)
    logp = torch.where(kept, (x.gather(1, at) - lse).view(-1), 0.0)
    if st["case"]["train"]:
        w = torch.where(kept, st["weights"], 0.0).view(-1, 1)
        grad = (e / s) * -w
        grad.scatter_add_(1, at, w)
        return logp, grad.to(st["logits"].dtype)
    entropy = (torch.log(s) - (e * (x - m)).sum(dim=1, keepdim=True) / s).view(-1)
    k = st["case"]["top"]
    if k == 0:
        return logp, entropy
    # the largest logits one after another, the lowest index among equals
    index = torch.arange(V, device=x.device)
    ids, vals = [], []
    for _ in range(k):
        m = x.max(dim=1, keepdim=True).values
        i = torch.where(x == m, index, V).min(dim=1, keepdim=True).values
        ids.append(i)
        vals.append(m - lse)
        x = x.scatter(1, i, -math.inf)
    return logp, entropy, torch.cat(vals, dim=1), torch.cat(ids, dim=1)


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "adapters":
        return _exact_adapters(case, st)
    if case["op"] == "embed":
        return _exact_embed(case, st)
    return _exact_logprobs(case, st)


def _exact_adapters(case, st):
    s = st["scale"]
    pieces_y, pieces_dx = [], []
    n, r, K, M = case["clients"], case["rank"], case["k"], case["m"]
    grads = torch.zeros(n, r * K + M * r, dtype=torch.float64, device="cuda") if case["train"] else None
    for (a, b, c) in _segments(st):
        xs = st["x"][a:b].double()
        Ac, Bc = st["A"][c].double(), st["B"][c].double()
        hidden = torch.matmul(xs, Ac.T.contiguous())
        delta = torch.matmul(hidden, Bc.T.contiguous())
        pieces_y.append(st["base"][a:b].double() + s * delta)
        if case["train"]:
            ds = st["dy"][a:b].double() * s
            z = torch.matmul(ds, Bc)
            pieces_dx.append(st["dx_base"][a:b].double() + torch.matmul(z, Ac))
            grads[c, :r * K] = torch.matmul(z.T.contiguous(), xs).reshape(-1)
            grads[c, r * K:] = torch.matmul(ds.T.contiguous(), hidden).reshape(-1)
    y = torch.cat(pieces_y)
    return (y, torch.cat(pieces_dx), grads) if case["train"] else y


def _exact_embed(case, st):
    outs = []
    n, V, E = case["clients"], case["vocab"], case["dim"]
    grad = torch.zeros(n, V, E, dtype=torch.float64, device="cuda") if case["train"] else None
    for (a, b, c) in _segments(st):
        ids = st["ids"][a:b]
        outs.append(st["table"][c][ids].double() * st["scale"])
        if case["train"]:
            order = torch.argsort(ids, stable=True)
            sums = torch.cumsum(st["dy"][a:b][order].double(), dim=0)
            seen, counts = torch.unique_consecutive(ids[order], return_counts=True)
            last = torch.cumsum(counts, 0) - 1
            totals = sums[last]
            totals[1:] -= sums[last[:-1]]
            grad[c, seen] = totals * st["scale"]
    out = torch.cat(outs)
    return (out, grad) if case["train"] else out


def _exact_logprobs(case, st):
    cols = [[], [], [], []]
    V, k = case["vocab"], case["top"]
    step = max(1, (1 << 27) // V)
    for a in range(0, case["rows"], step):
        x = st["logits"][a:a + step].double()
        t = st["targets"][a:a + step]
        logp = x - torch.logsumexp(x, dim=1, keepdim=True)
        safe = t.clamp(min=0)
        picked = logp[torch.arange(len(t), device="cuda"), safe]
        cols[0].append(torch.where(t >= 0, picked, torch.zeros_like(picked)))
        p = torch.exp(logp)
        if case["train"]:
            d = p.neg_()
            d[torch.arange(len(t), device="cuda"), safe] += 1.0
            cols[1].append(d * torch.where(t >= 0, st["weights"][a:a + step], 0.0).double().view(-1, 1))
            continue
        cols[1].append(-(p * logp).sum(dim=1))
        if k:
            for j in range(0, len(t), 64):       # a stable descending sort keeps the lowest index first
                v, i = torch.sort(logp[j:j + 64], dim=1, descending=True, stable=True)
                cols[2].append(v[:, :k].clone())
                cols[3].append(i[:, :k].clone())
    return tuple(torch.cat(c) for c in cols if c)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    e = _SIZE[case["dtype"]]
    if case["op"] == "adapters":
        T, K, M, r = case["tokens"], case["k"], case["m"], case["rank"]
        weights = case["segments"] * r * (K + M) * _SIZE[case["weights"]]
        nbytes = T * (K + 2 * M) * e + weights
        flops = 2 * T * r * (K + M)
        if case["train"]:
            nbytes += T * (2 * K + M) * e + case["clients"] * r * (K + M) * 4
            flops *= 3
        return {"bytes": nbytes, "flops": flops}
    if case["op"] == "embed":
        T, V, E = case["tokens"], case["vocab"], case["dim"]
        # rows of the tables that the skewed ids reach, each read once
        rank = torch.arange(1, V + 1, dtype=torch.float64)
        p = torch.log1p(1 / rank) / math.log(V + 1)
        reached = float((1 - (1 - p) ** (T / case["clients"])).sum()) * case["clients"]
        nbytes = T * 8 + T * E * e + int(reached) * E * 4
        flops = T * E
        if case["train"]:
            nbytes += T * E * e + case["clients"] * V * E * 4
            flops += T * E
        return {"bytes": nbytes, "flops": flops}
    T, V = case["rows"], case["vocab"]
    nbytes = T * V * e * (2 if case["train"] else 1) + T * 12
    return {"bytes": nbytes, "flops": T * V * (5 if case["train"] else 4)}

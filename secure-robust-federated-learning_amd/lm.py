"""Operators of clients that are language models, for all clients of a round at
once (libsra.so, include/sra.h k12-k14).

The reference trains its clients one after another (src/simulate.py:150-202);
these let one batch hold the tokens of every client and read or write rows of
the clients' (N, D) matrices (``store.ClientBank``):

* ``adapter_apply`` / ``adapter_grad`` -- every client's low-rank adapter beside
  a shared projection, and its gradients;
* ``embed`` / ``embed_grad`` -- embedding lookup with scaling from one shared
  table or one table a client, and the table's gradient by sorted tokens;
* ``token_logprobs`` / ``token_logprobs_and_grad`` / ``token_logprobs_grad`` --
  log probabilities of given tokens with entropy and top alternatives (the loss
  and accuracy of simulate.py:407-459 come from them), and the logits' gradient;
* ``adapters`` / ``embedding`` / ``token_logp`` -- the same for torch.autograd.

``offsets`` (int64, S + 1 ascending values) and ``slots`` (int32, S) are device
tensors: tokens [offsets[s], offsets[s + 1]) belong to row ``slots[s]`` of the
clients' matrices, -1 for none; tokens no segment covers have none either.  They
are read on the device only, so a captured graph replays with new values.  A
slot or token id outside its range is treated as none and counted, once a token
and call (``engine.row_fault_count``).

Everything runs on torch's current stream of the tensors' device and allocates
through torch's caching allocator.  Tensors given to be written (``out`` and the
like) get a new version, as torch's own in-place operations give.  There is no CPU
path.

Inputs that the kernels cannot walk (columns apart, matrices of a slot that are not
contiguous) are copied on every call: 8 tables of 17 MB, transposed in memory, make a
lookup of 11 us one of 140 us.
"""
from __future__ import annotations

import functools
from collections import namedtuple

import torch

from . import _lib

MAX_RANK = 64
MAX_TOP = 32
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


class TokenLogprobs(namedtuple("TokenLogprobs", "logp entropy lse top_logp top_ids")):
    """Beside the five: ``lse_rest``, what the rounding of lse left."""

    lse_rest = None



# ---------------------------------------------------------------------------
# argument checks: the usual tensors (contiguous, of the expected shape) pass on
# the first line of each, the small calls are bound by this code
# ---------------------------------------------------------------------------
def _device_tensor(name, t, device=None):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError("%s must be a CUDA (HIP) tensor, got %r" % (name, type(t)))
    if device is not None and t.device != device:
        raise ValueError("%s is on %s, expected %s" % (name, t.device, device))
    return t


def _float_code(name, t):
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise TypeError("%s must be float32, bfloat16 or float16, got %s" % (name, t.dtype))
    return code


def _check(name, t, shape, dtype, device):
    _device_tensor(name, t, device)
    if t.shape != shape:
        raise ValueError("%s must have shape %s, got %s" % (name, tuple(shape), tuple(t.shape)))
    if dtype is not None and t.dtype is not dtype:
        raise TypeError("%s must be %s, got %s" % (name, dtype, t.dtype))


def _rows(name, t, shape, dtype, device, out=False):
    """A matrix the kernels can walk as row * stride + column, and that stride.
    Inputs whose columns are strided or whose rows overlap are copied; outputs are
    refused."""
    _check(name, t, shape, dtype, device)
    r, c = shape
    if t.is_contiguous():
        return t, c
    s0, s1 = t.stride()
    if (c > 1 and s1 != 1) or (r > 1 and s0 < c):
        if out:
            raise ValueError("%s needs unit column stride and rows that do not overlap" % name)
        return t.contiguous(), c
    return t, (s0 if r > 1 else c)


def _slot_rows(name, t, shape, device, dtype=None, out=False):
    """(n, *matrix) whose matrices are contiguous, and the slot stride."""
    _check(name, t, shape, dtype, device)
    n, a, b = shape
    if t.is_contiguous():
        return t, a * b
    s0, s1, s2 = t.stride()
    if (a > 1 and s1 != b) or (b > 1 and s2 != 1) or (n > 1 and s0 < a * b):
        if out:
            raise ValueError("%s needs contiguous slots that do not overlap" % name)
        return t.contiguous(), a * b
    return t, (s0 if n > 1 else a * b)


def _vector(name, t, n, dtype, device):
    _check(name, t, (n,), dtype, device)
    return t if t.is_contiguous() else t.contiguous()


def _segments(offsets, slots, device):
    if offsets is None or slots is None:
        raise ValueError("offsets and slots go together")
    _device_tensor("slots", slots, device)
    if slots.dim() != 1:
        raise ValueError("slots must be a vector, got shape %s" % (tuple(slots.shape),))
    n = slots.shape[0]
    return (_vector("offsets", offsets, n + 1, torch.int64, device), _vector("slots", slots, n, torch.int32, device), n)


def _ptr(t):
    return t.data_ptr() if t is not None else None


# absent from a torch without GPU support, whose tensors are refused before it is needed
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _call(device, name, *args):
    """One library call on the device's current stream (the last argument)."""
    index = device.index
    if index == torch.cuda.current_device():
        _lib.call(name, *args, _raw_stream(index))
    else:
        with torch.cuda.device(device):
            _lib.call(name, *args, _raw_stream(index))


# The kernels write behind torch's back: the caller's tensors get a new version, so
# that autograd refuses a backward pass through what it saved before.
_written = torch.autograd.graph.increment_version


@functools.lru_cache(maxsize=4096)
def _bytes(name, *args):
    """A workspace size: a function of the sizes alone."""
    return _lib.query_bytes(name, *args)


# ---------------------------------------------------------------------------
# k12: low-rank adapters beside a shared projection
# ---------------------------------------------------------------------------
def _adapter_args(x, A, B, offsets, slots):
    _device_tensor("x", x)
    if x.dim() != 2 or not isinstance(A, torch.Tensor) or not isinstance(B, torch.Tensor) or A.dim() != 3 \
            or B.dim() != 3:
        raise ValueError("x must be (tokens, k), A (slots, rank, k) and B (slots, m, rank)")
    dtype = _float_code("x", x)
    T, K = x.shape
    n, r, _ = A.shape
    M = B.shape[1]
    if r < 1 or n < 1 or K < 1 or M < 1:
        raise ValueError("adapters need at least one slot, rank, input and output, got A %s, B %s"
                         % (tuple(A.shape), tuple(B.shape)))
    if r > MAX_RANK:
        raise NotImplementedError("adapter rank %d is above %d" % (r, MAX_RANK))
    if A.dtype != B.dtype or A.dtype not in (torch.float32, x.dtype):
        raise TypeError("A and B must both be float32 or %s, got %s and %s" % (x.dtype, A.dtype, B.dtype))
    A, lda = _slot_rows("A", A, (n, r, K), x.device)
    B, ldb = _slot_rows("B", B, (n, M, r), x.device)
    x, ldx = _rows("x", x, (T, K), x.dtype, x.device)
    offsets, slots, S = _segments(offsets, slots, x.device)
    head = (x.data_ptr(), ldx, A.data_ptr(), lda, B.data_ptr(), ldb, offsets.data_ptr(), slots.data_ptr(), S, T, n, K,
            M, r)
    keep = (x, A, B, offsets, slots)
    return head, keep, T, K, M, n, r, dtype, _DTYPES[A.dtype]


def _adapter_workspace(T, S, n, K, M, r, device):
    nb = _bytes("sra_adapter_workspace_bytes", T, S, n, K, M, r)
    return torch.empty(nb, dtype=torch.uint8, device=device), nb


def adapter_apply(base, x, A, B, offsets, slots, scale=1.0, out=None, hidden=False):
    """``out[t] = base[t] + scale * B[c] @ (A[c] @ x[t])`` for the tokens t of slot c.

    x (T, K) and base (T, M) are activations of one type (float32, bfloat16,
    float16); base None means zeros.  A (n, r, K) and B (n, M, r) are float32 (rows
    of the clients' matrix) or the activations' type, 1 <= r <= 64.  Tokens without
    a slot get base.  An infinite operand makes its products infinite or NaN.
    ``out`` may be base (in place).  hidden=True also returns the
    float32 (T, r) products A x for ``adapter_grad``."""
    head, keep, T, K, M, n, r, dtype, wdtype = _adapter_args(x, A, B, offsets, slots)
    dev = x.device
    ldbase = M
    if base is not None:
        base, ldbase = _rows("base", base, (T, M), x.dtype, dev)
    ldo = M
    given = out is not None
    if not given:
        out = torch.empty((T, M), dtype=x.dtype, device=dev)
    else:
        out, ldo = _rows("out", out, (T, M), x.dtype, dev, out=True)
    H = torch.empty((T, r), dtype=torch.float32, device=dev) if hidden else None
    ws, nb = _adapter_workspace(T, slots.shape[0], n, K, M, r, dev)
    _call(dev, "sra_adapter_apply", _ptr(base), ldbase, *head, float(scale), dtype, wdtype, out.data_ptr(), ldo,
          _ptr(H), ws.data_ptr(), nb)
    if given:
        _written(out)
    return (out, H) if hidden else out


def adapter_grad(grad_out, x, A, B, offsets, slots, scale=1.0, hidden=None, base_grad=None, grad_x=True, grad_A=True,
                 grad_B=True, accumulate=False):
    """Gradients of ``adapter_apply``: (dx, dA, dB).

    dx = base_grad + scale * A' B' grad_out (x's type; base_grad, the shared
    projection's part, None for zeros); dA (n, r, K) and dB (n, M, r) are float32.
    Each of grad_x, grad_A, grad_B is True (a new tensor), False (None returned) or
    the tensor to write; grad_x may be base_grad, but not grad_out or x.  Every slot
    of dA and dB is written, zeros where it has no token; accumulate=True adds to the
    tensors given instead.  ``hidden`` is adapter_apply's, or None to compute it
    again."""
    head, keep, T, K, M, n, r, dtype, wdtype = _adapter_args(x, A, B, offsets, slots)
    dev = x.device
    dy, lddy = _rows("grad_out", grad_out, (T, M), x.dtype, dev)
    if accumulate and (grad_A is True or grad_B is True):
        raise ValueError("accumulate=True needs the grad_A and grad_B to add to")
    if hidden is not None:
        hidden, _ = _rows("hidden", hidden, (T, r), torch.float32, dev)
        hidden = hidden.contiguous()
    lddxb = K
    if base_grad is not None:
        base_grad, lddxb = _rows("base_grad", base_grad, (T, K), x.dtype, dev)

    def target(name, t, make, check):
        if t is False or t is None:
            return None, 0
        return check(name, make() if t is True else t)

    dx, lddx = target("grad_x", grad_x, lambda: torch.empty((T, K), dtype=x.dtype, device=dev),
                      lambda a, t: _rows(a, t, (T, K), x.dtype, dev, out=True))
    dA, ldda = target("grad_A", grad_A, lambda: torch.empty((n, r, K), dtype=torch.float32, device=dev),
                      lambda a, t: _slot_rows(a, t, (n, r, K), dev, torch.float32, out=True))
    dB, lddb = target("grad_B", grad_B, lambda: torch.empty((n, M, r), dtype=torch.float32, device=dev),
                      lambda a, t: _slot_rows(a, t, (n, M, r), dev, torch.float32, out=True))
    ws, nb = _adapter_workspace(T, slots.shape[0], n, K, M, r, dev)
    _call(dev, "sra_adapter_grad", dy.data_ptr(), lddy, *head, float(scale), dtype, wdtype, _ptr(hidden),
          _ptr(base_grad), lddxb, _ptr(dx), lddx, _ptr(dA), ldda, _ptr(dB), lddb, int(bool(accumulate)),
          ws.data_ptr(), nb)
    for asked, t in ((grad_x, dx), (grad_A, dA), (grad_B, dB)):
        if t is not None and asked is not True:
            _written(t)
    return dx, dA, dB


# ---------------------------------------------------------------------------
# k13: embedding
# ---------------------------------------------------------------------------
def _table(name, table, offsets, slots, out=False):
    """(pointer owner, slot stride, n, V, E, segments) of a (V, E) table for every
    token or (n, V, E) tables of n slots."""
    _device_tensor(name, table)
    if table.dim() not in (2, 3) or 0 in table.shape:
        raise ValueError("%s must be a (vocab, dim) or (slots, vocab, dim) tensor, got %s"
                         % (name, tuple(table.shape)))
    if offsets is None and slots is None:
        if table.dim() == 3:
            raise ValueError("%s of %d slots needs offsets and slots" % (name, table.shape[0]))
        seg = (None, None, 0)
    else:
        if table.dim() == 2:
            raise ValueError("offsets and slots need a (slots, vocab, dim) tensor; use %s[None]" % name)
        seg = _segments(offsets, slots, table.device)
    full = table if table.dim() == 3 else table[None]
    full, ld = _slot_rows(name, full, full.shape, table.device, out=out)
    n, V, E = full.shape
    return full, ld, n, V, E, seg


def embed(table, ids, offsets=None, slots=None, scale=1.0, dtype=None, out=None):
    """``out[t] = scale * table[ids[t]]`` for one shared (V, E) table, or
    ``scale * table[c][ids[t]]`` for the tokens t of slot c of an (n, V, E) one.

    The product is formed in float32 and rounded once to ``dtype`` (the table's by
    default).  ids (T,) are int64.  Tokens without a slot, or with an id outside
    the vocabulary (counted), get zeros.  ``out`` must not be the table."""
    full, ld, n, V, E, (off, sl, S) = _table("table", table, offsets, slots)
    code = _float_code("table", full)
    dev = full.device
    ids = _vector("ids", _device_tensor("ids", ids, dev), ids.numel(), torch.int64, dev)
    T = ids.shape[0]
    given = out is not None
    if not given:
        out = torch.empty((T, E), dtype=dtype or full.dtype, device=dev)
    elif dtype is not None and out.dtype != dtype:
        raise TypeError("out must be %s, got %s" % (dtype, out.dtype))
    out, ldo = _rows("out", out, (T, E), None, dev, out=True)
    _call(dev, "sra_embed", full.data_ptr(), ld, code, ids.data_ptr(), _ptr(off), _ptr(sl), S, T, n, V, E,
          float(scale), out.data_ptr(), ldo, _float_code("out", out))
    if given:
        _written(out)
    return out


def embed_grad(grad_out, ids, grad, offsets=None, slots=None, scale=1.0, padding_idx=None, accumulate=False):
    """The table's gradient into ``grad`` (float32, (V, E) or (n, V, E) like the
    table): ``grad[c][v] = scale * sum of grad_out[t]`` over slot c's tokens with
    ids[t] = v, summed in float32, t ascending, without atomics.

    Tokens with ids[t] = padding_idx add nothing.  Every row is written, zeros
    where no token reads it; accumulate=True adds to the rows that tokens read and
    leaves the others alone.  ``grad`` must not be grad_out."""
    full, ld, n, V, E, (off, sl, S) = _table("grad", grad, offsets, slots, out=True)
    dev = full.device
    if full.dtype != torch.float32:
        raise TypeError("grad must be float32, got %s" % full.dtype)
    ids = _vector("ids", _device_tensor("ids", ids, dev), ids.numel(), torch.int64, dev)
    T = ids.shape[0]
    dy, lddy = _rows("grad_out", grad_out, (T, E), None, dev)
    code = _float_code("grad_out", dy)
    pad = -1
    if padding_idx is not None:
        pad = int(padding_idx)
        if not 0 <= pad < V:
            raise ValueError("padding_idx must be in [0, %d), got %d" % (V, pad))
    nb = _bytes("sra_embed_grad_workspace_bytes", T, E)
    ws = torch.empty(nb, dtype=torch.uint8, device=dev)
    _call(dev, "sra_embed_grad", dy.data_ptr(), lddy, code, ids.data_ptr(), _ptr(off), _ptr(sl), S, T, n, V, E,
          float(scale), pad, full.data_ptr(), ld, int(bool(accumulate)), ws.data_ptr(), nb)
    _written(grad)
    return grad


# ---------------------------------------------------------------------------
# k14: log probabilities of given tokens
# ---------------------------------------------------------------------------
def _logits(logits, targets):
    _device_tensor("logits", logits)
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError("logits must be (rows, vocab), got %s" % (tuple(logits.shape),))
    code = _float_code("logits", logits)
    logits, ldl = _rows("logits", logits, logits.shape, logits.dtype, logits.device)
    targets = _vector("targets", targets, logits.shape[0], torch.int64, logits.device)
    return logits, ldl, code, targets


def _logprobs(logits, targets, top, entropy, ignore_index, grad_logp, grad_entropy, out):
    src = logits
    logits, ldl, code, targets = _logits(logits, targets)
    R, V = logits.shape
    dev = logits.device
    top = int(top)
    if not 0 <= top <= V:
        raise ValueError("top must be in [0, %d], got %d" % (V, top))
    if top > MAX_TOP:
        raise NotImplementedError("top %d is above %d" % (top, MAX_TOP))

    # logp, lse and the alternatives come as views of one buffer
    f = torch.empty((3 + bool(entropy) + top) * R, dtype=torch.float32, device=dev)
    rows = f[:(3 + bool(entropy)) * R].view(3 + bool(entropy), R).unbind(0)
    res = TokenLogprobs(rows[0], rows[3] if entropy else None, rows[1], f[(3 + bool(entropy)) * R:].view(R, top),
                        torch.empty((R, top), dtype=torch.int64, device=dev))
    res.lse_rest = rows[2]
    grad, ldg, given = None, 0, out is not None
    if grad_logp is not None:
        grad_logp = _vector("grad_logp", grad_logp, R, torch.float32, dev)
        if grad_entropy is not None:
            grad_entropy = _vector("grad_entropy", grad_entropy, R, torch.float32, dev)
        if out is src and logits is not src:
            raise ValueError("out can be the logits only where they have unit column stride")
        if out is None:
            out = torch.empty((R, V), dtype=logits.dtype, device=dev)
        grad, ldg = _rows("out", out, (R, V), logits.dtype, dev, out=True)
    _call(dev, "sra_token_logprobs_split", logits.data_ptr(), ldl, code, targets.data_ptr(), R, V, int(ignore_index),
          top, res.logp.data_ptr(), _ptr(res.entropy), res.lse.data_ptr(), res.lse_rest.data_ptr(),
          res.top_logp.data_ptr(), res.top_ids.data_ptr(), _ptr(grad_logp), _ptr(grad_entropy), _ptr(grad), ldg)
    if given:
        _written(grad)
    return res, grad


def token_logprobs(logits, targets, top=0, entropy=False, ignore_index=-100):
    """TokenLogprobs(logp, entropy, lse, top_logp, top_ids) of (rows, vocab) logits.

    logp[r] = log softmax(logits[r])[targets[r]] (float32; 0 where the target is
    ignore_index, NaN and counted where it is outside the vocabulary); entropy of
    every row when asked, else None; lse the log of the sum of exponentials; the
    ``top`` <= 32 most probable tokens' log probabilities and ids, descending, the
    lowest id first among equals.  -inf logits have probability 0; a row of only
    -inf (lse -inf), or with +inf or NaN, gives NaN.  ``lse_rest`` of the result is
    what the rounding of lse left, for ``token_logprobs_grad``."""
    return _logprobs(logits, targets, top, entropy, ignore_index, None, None, None)[0]


def token_logprobs_and_grad(logits, targets, grad_logp, grad_entropy=None, top=0, entropy=False, ignore_index=-100,
                            out=None):
    """``token_logprobs`` and the logits' gradient for given row gradients of logp
    and entropy (float32 (rows,)), in one pass over the logits up to a vocabulary of
    65536 (float32: 32768), in two beyond: a mean loss over n targets is
    grad_logp = -1 / n.  Rows with an ignored or bad target, or with grad_logp 0, get
    zeros (beside the entropy's part) whatever their logits are.  ``out`` may be the
    logits (in place)."""
    if grad_logp is None:
        raise ValueError("grad_logp is needed")
    return _logprobs(logits, targets, top, entropy, ignore_index, grad_logp, grad_entropy, out)


def token_logprobs_grad(logits, targets, lse, grad_logp, entropy=None, grad_entropy=None, ignore_index=-100, out=None,
                        lse_rest=None):
    """The logits' gradient from a forward pass's lse and lse_rest (and entropy, which
    grad_entropy needs).  Without lse_rest every probability of a row is off by up to
    2^-24 |lse| of itself.  ``out`` may be the logits (in place)."""
    src = logits
    logits, ldl, code, targets = _logits(logits, targets)
    R, V = logits.shape
    dev = logits.device
    lse = _vector("lse", lse, R, torch.float32, dev)
    if lse_rest is not None:
        lse_rest = _vector("lse_rest", lse_rest, R, torch.float32, dev)
    grad_logp = _vector("grad_logp", grad_logp, R, torch.float32, dev)
    if grad_entropy is not None:
        if entropy is None:
            raise ValueError("grad_entropy needs the forward pass's entropy")
        grad_entropy = _vector("grad_entropy", grad_entropy, R, torch.float32, dev)
        entropy = _vector("entropy", entropy, R, torch.float32, dev)
    if out is src and logits is not src:
        raise ValueError("out can be the logits only where they have unit column stride")
    given = out is not None
    if not given:
        out = torch.empty((R, V), dtype=logits.dtype, device=dev)
    out, ldg = _rows("out", out, (R, V), logits.dtype, dev, out=True)
    _call(dev, "sra_token_logprobs_grad_split", logits.data_ptr(), ldl, code, targets.data_ptr(), R, V,
          int(ignore_index), lse.data_ptr(), _ptr(lse_rest), _ptr(entropy), grad_logp.data_ptr(), _ptr(grad_entropy), out.data_ptr(), ldg)
    if given:
        _written(out)
    return out


# ---------------------------------------------------------------------------
# torch.autograd
# ---------------------------------------------------------------------------
def _not_capturing(*tensors):
    """autograd's leaf accumulation belongs to the stream a leaf was first used
    on: under capture it would tie an eager graph to the captured one."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors) \
            and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("the autograd forms cannot be captured into a graph; capture adapter_apply / adapter_grad, "
                           "embed / embed_grad and token_logprobs / token_logprobs_grad")


class _Adapters(torch.autograd.Function):
    @staticmethod
    def forward(ctx, base, x, A, B, offsets, slots, scale):
        y, hidden = adapter_apply(base, x, A, B, offsets, slots, scale, hidden=True)
        ctx.save_for_backward(x, A, B, offsets, slots, hidden)
        ctx.scale = scale
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, A, B, offsets, slots, hidden = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, dA, dB = adapter_grad(dy, x, A, B, offsets, slots, ctx.scale, hidden, grad_x=need[1], grad_A=need[2],
                                  grad_B=need[3])
        return (dy if need[0] else None, dx, dA.to(A.dtype) if need[2] else None,
                dB.to(B.dtype) if need[3] else None, None, None, None)


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, ids, offsets, slots, scale, padding_idx, dtype):
        ctx.save_for_backward(ids, offsets, slots)
        ctx.args = (tuple(table.shape), table.dtype, scale, padding_idx)
        return embed(table, ids, offsets, slots, scale, dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        ids, offsets, slots = ctx.saved_tensors
        shape, dtype, scale, padding_idx = ctx.args
        grad = torch.empty(shape, dtype=torch.float32, device=dy.device)
        embed_grad(dy, ids, grad, offsets, slots, scale, padding_idx)
        return grad.to(dtype), None, None, None, None, None, None


class _TokenLogp(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, ignore_index):
        res = token_logprobs(logits, targets, entropy=True, ignore_index=ignore_index)
        ctx.save_for_backward(logits, targets, res.lse, res.lse_rest, res.entropy)
        ctx.ignore_index = ignore_index
        return res.logp, res.entropy

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dlogp, dent):
        logits, targets, lse, rest, ent = ctx.saved_tensors
        return token_logprobs_grad(logits, targets, lse, dlogp, ent, dent, ctx.ignore_index, lse_rest=rest), None, None


def adapters(base, x, A, B, offsets, slots, scale=1.0):
    """``adapter_apply`` with gradients for base, x, A and B."""
    _not_capturing(base, x, A, B)
    return _Adapters.apply(base, x, A, B, offsets, slots, float(scale))


def embedding(table, ids, offsets=None, slots=None, scale=1.0, padding_idx=None, dtype=None):
    """``embed`` with a gradient for the table."""
    _not_capturing(table)
    return _Embedding.apply(table, ids, offsets, slots, float(scale), padding_idx, dtype)


def token_logp(logits, targets, ignore_index=-100):
    """(logp, entropy) of ``token_logprobs`` with gradients for the logits."""
    _not_capturing(logits)
    return _TokenLogp.apply(logits, targets, int(ignore_index))


def evaluate(logits, targets, ignore_index=-100):
    """(summed loss, correct predictions, counted targets) of a batch as device
    scalars: what simulate.py:407-459 adds up for the results row's test loss and
    accuracy (``formats.format_result_row``)."""
    res = token_logprobs(logits, targets, top=1, ignore_index=ignore_index)
    kept = targets != ignore_index
    return -res.logp.sum(), ((res.top_ids[:, 0] == targets) & kept).sum(), kept.sum()

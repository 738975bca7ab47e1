"""Refusals of the language-model client operators: what the C ABI and the
Python entry points turn into errors before anything reaches a GPU."""
from __future__ import annotations

import ctypes

import pytest
import torch

from srfl_amd import _lib, lm

P = ctypes.c_void_p(4096)      # never dereferenced: validation fails first
BIG = 1 << 30


def adapter_args(**kw):
    a = dict(base=P, ldbase=64, x=P, ldx=64, A=P, lda=512, B=P, ldb=512, offsets=P, slots=P, nseg=2, tokens=8, nslots=4,
             k=64, m=64, rank=8, scale=1.0, dtype=1, wdtype=0, out=P, ldo=64, hidden=None, ws=P, ws_bytes=BIG)
    a.update(kw)
    return list(a.values()) + [None]


@pytest.mark.parametrize("kw,exc,match", [
    (dict(x=None), ValueError, "non-null"), (dict(out=None), ValueError, "non-null"),
    (dict(offsets=None), ValueError, "offsets"), (dict(slots=None), ValueError, "slots"),
    (dict(rank=0), ValueError, "rank"), (dict(rank=65), NotImplementedError, "rank"),
    (dict(k=0), ValueError, "k and m"), (dict(m=-1), ValueError, "k and m"), (dict(tokens=-1), ValueError, "tokens"),
    (dict(tokens=1 << 31), ValueError, "tokens"), (dict(nslots=0), ValueError, "nslots"),
    (dict(dtype=3), ValueError, "dtype"), (dict(wdtype=2), ValueError, "wdtype"),
    (dict(dtype=0, wdtype=1), ValueError, "wdtype"),
    (dict(ldx=63), ValueError, "stride"), (dict(ldo=63), ValueError, "stride"), (dict(ldbase=63), ValueError, "stride"),
    (dict(lda=511), ValueError, "slot strides"), (dict(ldb=511), ValueError, "slot strides"),
    (dict(ws_bytes=8), ValueError, "workspace"), (dict(ws=None), ValueError, "workspace"),
    (dict(nseg=-1), ValueError, "nseg"),
    (dict(ldbase=65), ValueError, "one buffer"),          # base and out are the same pointer here
])
def test_adapter_apply_refuses(kw, exc, match):
    with pytest.raises(exc, match=match):
        _lib.call("sra_adapter_apply", *adapter_args(**kw))


def test_adapter_workspace_refuses():
    with pytest.raises(NotImplementedError):
        _lib.query_bytes("sra_adapter_workspace_bytes", 8, 1, 1, 64, 64, 65)
    with pytest.raises(ValueError):
        _lib.query_bytes("sra_adapter_workspace_bytes", 8, 1, 1, 0, 64, 8)


@pytest.mark.parametrize("kw,exc,match", [
    (dict(dout=None), ValueError, "dout"), (dict(lddo=63), ValueError, "stride"), (dict(lddx=63), ValueError, "stride"),
    (dict(ldda=511), ValueError, "slot strides"), (dict(lddb=511), ValueError, "slot strides"),
    (dict(rank=65), NotImplementedError, "rank"), (dict(ws_bytes=8), ValueError, "workspace"),
    (dict(lddxb=70), ValueError, "one buffer"), (dict(nslots=65536), NotImplementedError, "65535"),
])
def test_adapter_grad_refuses(kw, exc, match):
    a = dict(dout=P, lddo=64, x=P, ldx=64, A=P, lda=512, B=P, ldb=512, offsets=P, slots=P, nseg=2, tokens=8, nslots=4,
             k=64, m=64, rank=8, scale=1.0, dtype=1, wdtype=0, hidden=None, dxbase=P, lddxb=64, dx=P, lddx=64, dA=P,
             ldda=512, dB=P, lddb=512, accumulate=0, ws=P, ws_bytes=BIG)
    a.update(kw)
    with pytest.raises(exc, match=match):
        _lib.call("sra_adapter_grad", *a.values(), None)


@pytest.mark.parametrize("kw,exc,match", [
    (dict(table=None), ValueError, "non-null"), (dict(ids=None), ValueError, "ids"),
    (dict(vocab=0), ValueError, "vocab"), (dict(dim=0), ValueError, "vocab"), (dict(dim=1 << 23), ValueError, "dim"),
    (dict(ldt=511), ValueError, "slot stride"), (dict(ldo=7), ValueError, "stride"),
    (dict(offsets=None, slots=None), ValueError, "offsets and slots"), (dict(slots=None), ValueError, "non-null"),
    (dict(tdtype=5), ValueError, "tdtype"), (dict(odtype=-1), ValueError, "odtype"),
])
def test_embed_refuses(kw, exc, match):
    a = dict(table=P, ldt=512, tdtype=0, ids=P, offsets=P, slots=P, nseg=2, tokens=8, nslots=4, vocab=64, dim=8,
             scale=1.0, out=P, ldo=8, odtype=1)
    a.update(kw)
    with pytest.raises(exc, match=match):
        _lib.call("sra_embed", *a.values(), None)


@pytest.mark.parametrize("kw,exc,match", [
    (dict(grad=None), ValueError, "non-null"), (dict(dout=None), ValueError, "non-null"),
    (dict(lddo=7), ValueError, "stride"), (dict(ldg=511), ValueError, "slot stride"),
    (dict(ws_bytes=8), ValueError, "workspace"),
    (dict(nslots=1 << 16, vocab=1 << 16, ldg=1 << 20), NotImplementedError, "2\\^32"),
])
def test_embed_grad_refuses(kw, exc, match):
    a = dict(dout=P, lddo=8, dtype=1, ids=P, offsets=P, slots=P, nseg=2, tokens=8, nslots=4, vocab=64, dim=8,
             scale=1.0, padding=-1, grad=P, ldg=512, accumulate=0, ws=P, ws_bytes=BIG)
    a.update(kw)
    with pytest.raises(exc, match=match):
        _lib.call("sra_embed_grad", *a.values(), None)


@pytest.mark.parametrize("kw,exc,match", [
    (dict(logits=None), ValueError, "non-null"), (dict(targets=None), ValueError, "non-null"),
    (dict(logp=None), ValueError, "non-null"), (dict(vocab=0), ValueError, "vocab"),
    (dict(vocab=1 << 28, ldl=1 << 28), ValueError, "vocab"), (dict(ldl=99), ValueError, "stride"),
    (dict(top=-1), ValueError, "top"), (dict(top=33), NotImplementedError, "top"),
    (dict(top=101, vocab=100), ValueError, "top"), (dict(top_ids=None), ValueError, "top"),
    (dict(grad_logp=None), ValueError, "grad_logp"), (dict(ldg=99), ValueError, "stride"),
    (dict(ldg=101), ValueError, "one buffer"), (dict(dtype=9), ValueError, "dtype"),
    (dict(logits=ctypes.c_void_p(4097)), ValueError, "aligned"),
])
def test_token_logprobs_refuses(kw, exc, match):
    a = dict(logits=P, ldl=100, dtype=1, targets=P, rows=4, vocab=100, ignore=-100, top=2, logp=P, entropy=P, lse=P,
             top_logp=P, top_ids=P, grad_logp=P, grad_entropy=None, grad=P, ldg=100)
    a.update(kw)
    with pytest.raises(exc, match=match):
        _lib.call("sra_token_logprobs", *a.values(), None)


def test_token_logprobs_grad_refuses():
    a = dict(logits=P, ldl=100, dtype=1, targets=P, rows=4, vocab=100, ignore=-100, lse=P, entropy=None, grad_logp=P,
             grad_entropy=P, grad=P, ldg=100)
    with pytest.raises(ValueError, match="entropy"):
        _lib.call("sra_token_logprobs_grad", *a.values(), None)
    a.update(grad_entropy=None, lse=None)
    with pytest.raises(ValueError, match="lse"):
        _lib.call("sra_token_logprobs_grad", *a.values(), None)


def test_python_entry_points_need_device_tensors():
    x = torch.zeros(4, 8)
    o, s = torch.tensor([0, 4]), torch.tensor([0], dtype=torch.int32)
    with pytest.raises(TypeError, match="CUDA"):
        lm.adapter_apply(x, x, torch.zeros(1, 2, 8), torch.zeros(1, 8, 2), o, s)
    with pytest.raises(TypeError, match="CUDA"):
        lm.embed(x, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(TypeError, match="CUDA"):
        lm.embed_grad(x, torch.zeros(4, dtype=torch.int64), torch.zeros(3, 8))
    with pytest.raises(TypeError, match="CUDA"):
        lm.token_logprobs(x, torch.zeros(4, dtype=torch.int64))
    with pytest.raises(ValueError, match="grad_logp"):
        lm.token_logprobs_and_grad(x, torch.zeros(4, dtype=torch.int64), None)


def test_zero_rows_and_tokens_need_no_launch():
    _lib.call("sra_adapter_apply", *adapter_args(tokens=0))
    _lib.call("sra_token_logprobs", None, 100, 1, None, 0, 100, -100, 0, None, None, None, None, None, None, None, None,
              0, None)
    _lib.call("sra_embed", P, 8, 0, None, None, None, 0, 0, 1, 4, 2, 1.0, None, 2, 0, None)


def test_launches_too_large_are_refused_before_any_kernel():
    """Counts that pass the checks of shapes but not what one launch holds."""
    many, ws = 1 << 30, 1 << 60
    with pytest.raises(NotImplementedError, match="too many"):
        _lib.call("sra_adapter_apply", *adapter_args(tokens=many, ws_bytes=ws))
    with pytest.raises(NotImplementedError, match="too many"):
        _lib.call("sra_adapter_apply", *adapter_args(tokens=1 << 25, k=4, m=4, rank=1, ws_bytes=ws))
    with pytest.raises(NotImplementedError, match="too many"):
        _lib.call("sra_embed", P, 512, 0, P, None, None, 0, many, 1, 64, 8, 1.0, P, 8, 1, None)
    with pytest.raises(NotImplementedError, match="too many"):
        _lib.call("sra_embed_grad", P, 4096, 1, P, None, None, 0, many, 1, 64, 4096, 1.0, -1, P, 1 << 18, 0, P, ws, None)
    with pytest.raises(NotImplementedError, match="too many"):
        _lib.call("sra_token_logprobs", P, 100, 1, P, many, 100, -100, 0, P, None, P, None, None, None, None, None, 0,
                  None)
    with pytest.raises(NotImplementedError, match="too many"):
        _lib.call("sra_token_logprobs_grad", P, 100, 1, P, many, 100, -100, P, None, P, None, P, 100, None)


@pytest.mark.parametrize("alias", ["dout", "x"])
def test_adapter_grad_refuses_dx_over_what_it_reads_later(alias):
    p = {q: ctypes.c_void_p(4096 * (i + 1)) for i, q in enumerate(("dout", "x", "dx"))}
    p["dx"] = p[alias]
    with pytest.raises(ValueError, match="dx must not be"):
        _lib.call("sra_adapter_grad", p["dout"], 64, p["x"], 64, P, 512, P, 512, P, P, 2, 8, 4, 64, 64, 8, 1.0, 1, 0,
                  None, None, 0, p["dx"], 64, P, 512, P, 512, 0, P, BIG, None)

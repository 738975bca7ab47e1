"""More refusals of the language-model operators, before anything reaches a GPU:
launches of empty batches, and outputs over inputs that are read after them."""
from __future__ import annotations

import ctypes

import pytest

from srfl_amd import _lib

P, Q = ctypes.c_void_p(4096), ctypes.c_void_p(8192)      # never dereferenced: validation fails first
BIG = 1 << 60


@pytest.mark.parametrize("which", ["dA", "dB"])
def test_gradients_of_an_empty_batch_too_large_for_a_launch(which):
    """Zeros for 64 * 2^27 values a slot would need 2^33 threads."""
    k, r = 1 << 27, 64
    a = dict(dout=P, lddo=k, x=P, ldx=k, A=P, lda=r * k, B=P, ldb=r * k, offsets=P, slots=P, nseg=2, tokens=0, nslots=1,
             k=k, m=k, rank=r, scale=1.0, dtype=1, wdtype=0, hidden=None, dxbase=None, lddxb=0, dx=None, lddx=0, dA=None,
             ldda=0, dB=None, lddb=0, accumulate=0, ws=P, ws_bytes=BIG)
    a.update({which: P, "ldd" + which[1]: r * k})
    with pytest.raises(NotImplementedError, match="too many"):
        _lib.call("sra_adapter_grad", *a.values(), None)


def test_embedding_gradient_over_the_gradient_it_reads():
    """The gradient is cleared before the tokens' gradients are read."""
    a = dict(dout=P, lddo=8, dtype=0, ids=Q, offsets=None, slots=None, nseg=0, tokens=64, nslots=1, vocab=64, dim=8,
             scale=1.0, padding=-1, grad=P, ldg=512, accumulate=0, ws=Q, ws_bytes=BIG)
    with pytest.raises(ValueError, match="grad must not be dout"):
        _lib.call("sra_embed_grad", *a.values(), None)


def test_lookup_over_its_table():
    a = dict(table=P, ldt=512, tdtype=0, ids=Q, offsets=None, slots=None, nseg=0, tokens=64, nslots=1, vocab=64, dim=8,
             scale=1.0, out=P, ldo=8, odtype=0)
    with pytest.raises(ValueError, match="out must not be the table"):
        _lib.call("sra_embed", *a.values(), None)

"""perf/operators.py: its plain forms and the framework's calls give the same
outputs on a state that is used again."""
from __future__ import annotations

import importlib.util
import os

import pytest
import torch

import lm_reference as ref

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "perf", "operators.py")


@pytest.fixture
def cases():
    spec = importlib.util.spec_from_file_location("lm_measured_cases", PATH)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("tokens,segments,k,m,rank", [(40, 3, 75, 61, 5), (300, 2, 128, 160, 16)])
def test_adapter_training_passes_on_one_state(cases, tokens, segments, k, m, rank, dtype):
    """Three passes of each side.  Both are within the bound of the formula, which
    three float32 passes over one buffer (the plain form's conversion of a float32
    dx_base is no copy) may use three times."""
    case = dict(op="adapters", train=True, tokens=tokens, segments=segments, clients=segments + 1, k=k, m=m, rank=rank,
                dtype=dtype, weights="fp32")
    got = []
    for own in (False, True):
        cases.own = own
        st = cases.prepare(case, 11)
        if not own:
            want = ref.adapter(st["base"], st["x"], st["A"], st["B"], st["host_offsets"], st["host_slots"], st["scale"],
                               st["x"].dtype, st["dy"], st["dx_base"])
        got.append([tuple(t.clone() for t in cases.run(st)) for _ in range(3)])
    for plain, own in zip(*got):
        ref.within("out", own[0], ref.d(plain[0]), 2 * want["out"][1])
        ref.within("dx", own[1], ref.d(plain[1]), 2 * 3 * want["dx"][1] + 6 * ref.U * ref.d(plain[1]).abs())
        n, split = case["clients"], rank * k
        bound = torch.cat([want["dA"][1].reshape(n, -1), want["dB"][1].reshape(n, -1)], dim=1)
        assert bound.shape[1] == split + m * rank
        ref.within("grads", own[2], ref.d(plain[2]), 2 * bound)

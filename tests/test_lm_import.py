"""The module of the language-model operators imports where torch has no GPU
support, and refuses CPU tensors there as anywhere."""
from __future__ import annotations

import importlib.util

import pytest
import torch

from srfl_amd import lm


def test_import_without_gpu_support(monkeypatch):
    monkeypatch.delattr(torch._C, "_cuda_getCurrentRawStream", raising=False)
    spec = importlib.util.spec_from_file_location("srfl_amd.lm_without_gpu", lm.__file__)
    bare = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(bare)
    with pytest.raises(TypeError, match="CUDA"):
        bare.token_logprobs(torch.zeros(2, 3), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(TypeError, match="CUDA"):
        bare.embed(torch.zeros(3, 4), torch.zeros(2, dtype=torch.int64))

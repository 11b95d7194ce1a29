"""Queries near the ends of bf16's range, where products run in f16: against keys and scales that bring the scores
back to an ordinary size (what 32 bits hold)."""
import numpy as np
import pytest
import torch

from test_gpu_kv import Setup, check_attend, queries


@pytest.fixture(autouse=True)
def _need_gpu():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("kv,exponent,size,scale", [("e4m3", -60, 1e17, 0.1), ("e4m3", -60, 5e37, 1e-20), ("e4m3", 110, 1e-33, None),
                                                    ("e4m3", 120, 1e-33, 2.0 ** -40), ("e4m3", 120, 1e-33, 2.0 ** -20),
                                                    ("f16", 0, 5e37, 1e-37), ("f16", 0, 1e-30, 1e30)])
def test_queries_of_any_size(kv, exponent, size, scale, rows):
    s = Setup([rows], [300], kv, 8, 2, 128, page=64, seed=8)
    s.ctx = s.lens
    s.fill()
    if kv == "e4m3":
        s.kv.k_scale.view(torch.uint8).fill_(127 + exponent)
    check_attend(s, queries(s, "bf16", size=size), "bf16", 1, scale=scale, rows=12)

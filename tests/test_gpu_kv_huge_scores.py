"""Attention whose scores pass 2^24 and more, where a score's own rounding is larger than 1."""
import numpy as np
import pytest
import torch

from test_gpu_kv import Setup


@pytest.fixture(autouse=True)
def _need_gpu():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["e4m3", "f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("size", [1e3, 1e6, 3e7, 1e10])
def test_huge_scores_stay_finite(kv, rows, size):
    """Scores of any size: a weight is at most the largest the products' type holds, where a reference's own steps are
    large too. Every output is an average of values."""
    s = Setup([rows], [300], kv, 8, 2, 128, page=64, seed=3)
    s.ctx = s.lens
    s.fill()
    g = torch.Generator(device="cuda").manual_seed(4)
    q = (size * torch.randn(rows, 8, 128, generator=g, device="cuda")).to(torch.bfloat16)
    out = s.kv.attend(0, q, s.batch, block_length=1).double().cpu().numpy()
    s.kv.check()
    v, _ = s.held("v", 0, s.lens[0])
    top = np.abs(v).max(0)[[h // 4 for h in range(8)]]
    assert np.isfinite(out).all() and (np.abs(out) <= top * (1 + 2.0 ** -6)).all()

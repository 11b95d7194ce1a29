"""Attention of zero and tiny queries over zero keys (a warm-up pass over zeros, padding): every visible position
weighs alike, whatever the number of rows, the mask and the page type."""
import numpy as np
import pytest
import torch

from test_gpu_kv import Setup, check_attend, queries


@pytest.fixture(autouse=True)
def _need_gpu():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["e4m3", "bf16", "f16"])
@pytest.mark.parametrize("rows", [1, 3, 64, 150])
@pytest.mark.parametrize("block", [1, 32])
def test_zero_queries_and_keys_give_the_mean_of_the_values(kv, rows, block):
    s = Setup([rows], [0], kv, 8, 2, 128, page=64, seed=rows)
    qkv = torch.randn(rows, 12 * 128, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    qkv[:, : 10 * 128] = 0.0
    w = torch.ones(128, device="cuda")
    q = s.kv.append(0, qkv, s.batch, n_head=8, q_norm=w, k_norm=w, rotary_dim=64, q_type=torch.bfloat16)
    assert not bool(q.any())
    check_attend(s, q, "bf16", block)
    qkv.zero_()
    s.kv.append(0, qkv, s.batch, n_head=8, q_norm=w, k_norm=w, rotary_dim=64, q_out=q)
    check_attend(s, q, "bf16", block)


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["e4m3", "f16"])
@pytest.mark.parametrize("rows", [1, 60])
@pytest.mark.parametrize("size,scale", [(0.0, None), (1e-30, None), (0.0, 1e-30), (1e-36, 1e-36)])
def test_tiny_queries_over_blocks_of_zero_keys(kv, rows, size, scale):
    """Some blocks of keys are zeros (of the smallest scale), some are not."""
    s = Setup([rows], [200], kv, 8, 2, 128, page=64, seed=7)
    s.ctx = s.lens
    s.fill()
    for p in range(0, s.lens[0], 32):
        if p // 32 % 2 or p + 32 >= s.lens[0]:
            pg, of = int(s.table[0, p // 64]), p % 64
            s.kv.k[0].view(torch.uint8 if kv == "e4m3" else torch.float16)[pg, :, of:of + 32] = 0
            if kv == "e4m3":
                s.kv.k_scale.view(torch.uint8)[0, pg, :, of // 32] = 127 - 60
    for block in (1, 32):
        check_attend(s, queries(s, "bf16", size=size), "bf16", block, scale=scale, rows=20)

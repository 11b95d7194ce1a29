"""A new cache's positions are zeros of the smallest scale: attention over positions that nothing has written yet
(a pass that warms up) gives zeros, and the logarithm of their number."""
import math

import pytest
import torch

import diffuse_moe as dm


@pytest.mark.gpu
@pytest.mark.parametrize("kv_type", ["e4m3", "bf16", "f16"])
@pytest.mark.parametrize("rows", [1, 4, 64])
def test_attention_over_a_new_cache(kv_type, rows):
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    kv = dm.PagedKV(n_pages=4, n_head_kv=2, head_dim=64, page_size=64, kv_type=kv_type)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    batch = kv.batch(i32([[3, 1, 0, 2]]), i32([0, rows]), i32([200]), rows)
    q = torch.randn(rows, 8, 64, device="cuda").to(torch.bfloat16)
    lse = torch.empty(rows, 8, device="cuda")
    out = kv.attend(0, q, batch, block_length=1, lse=lse)
    kv.check()
    assert not bool(out.any())
    want = torch.log(torch.arange(200 - rows + 1, 201, dtype=torch.float64, device="cuda"))[:, None].expand(rows, 8)
    assert bool(((lse.double() - want).abs() <= 2.0 ** -18 + math.log(200) * 2.0 ** -21).all())

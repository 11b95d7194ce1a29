"""Left padding so long that its elements pass 2^31 in eights: every padding row's query is zero."""
import pytest
import torch

import diffuse_moe as dm


@pytest.mark.gpu
def test_padding_past_31_bits():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    torch.cuda.empty_cache()
    heads, dim = 64, 128
    n = (1 << 31) // ((heads + 2) * dim // 8) + 5  # rows: their eights of elements, keys and values included, pass 2^31
    kv = dm.PagedKV(n_pages=1, n_head_kv=1, head_dim=dim, page_size=32, kv_type="bf16")
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    batch = kv.batch(i32([[0]]), i32([0, n]), i32([1]), n)
    qkv = torch.empty(n, (heads + 2) * dim, device="cuda", dtype=torch.float16)
    qkv[-1] = 1.0  # the one row that has a position
    q = torch.empty(n, heads, dim, device="cuda", dtype=torch.float16)
    for part in (q[:3], q[n // 2 - 1: n // 2 + 1], q[-3:]):
        part.fill_(7.0)
    kv.append(0, qkv, batch, n_head=heads, q_out=q)
    kv.check()
    for part in (q[:3], q[n // 2 - 1: n // 2 + 1], q[-3:-1]):
        assert not bool(part.any())
    assert bool((q[-1] == 1.0).all()) and bool((kv.k[0, 0, :, 0] == 1.0).all())
    del q, qkv
    torch.cuda.empty_cache()

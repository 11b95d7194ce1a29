"""Batches whose sequences overlap (a broken q_start) and so have more units of work than the host's check, which
counts every row once, allows for: reported, nothing computed."""
import numpy as np
import pytest
import torch

import diffuse_moe as dm


@pytest.mark.gpu
@pytest.mark.parametrize("n,heads", [(1024, 16), (1, 16)])
def test_overlapping_sequences_past_the_schedule(n, heads):
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    n_seq = 65536
    kv = dm.PagedKV(n_pages=1, n_head_kv=1, head_dim=64, page_size=65536, kv_type="e4m3")
    i32 = lambda a: torch.from_numpy(np.asarray(a, np.int32)).cuda()  # noqa: E731
    start = np.arange(n_seq + 1) % 2 * n  # 0, n, 0, n, ..: every other sequence has all n rows
    lens = np.full(n_seq, 1 << 20)
    batch = kv.batch(torch.zeros(n_seq, 16, dtype=torch.int32, device="cuda"), i32(start), i32(lens), n)
    q = torch.zeros(n, heads, 64, device="cuda", dtype=torch.bfloat16)
    out = torch.full_like(q, 7.0)
    if n == 1:  # the same tables with few units: positions 0 and 1 only
        batch.tensors[2].fill_(1)
    kv.attend(0, q, batch, out=out)
    with pytest.raises(dm.DmoeError, match="invalid q_start"):
        kv.check()
    assert n == 1 or bool((out == 7.0).all())

"""PagedKV.check() waits for the device: calls on any stream are heard."""
import pytest
import torch

import diffuse_moe as dm


@pytest.mark.gpu
def test_check_hears_calls_on_another_stream():
    kv = dm.PagedKV(n_pages=2, n_head_kv=2, head_dim=64, page_size=32, kv_type="e4m3")
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    batch = kv.batch(i32([[5]]), i32([0, 3]), i32([3]), 3)  # there is no page 5
    qkv = torch.randn(3, 8 * 64, device="cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)  # a tenth of a second
        kv.append(0, qkv, batch, n_head=4)
    with pytest.raises(dm.DmoeError, match="page number"):
        kv.check()
    kv.check()

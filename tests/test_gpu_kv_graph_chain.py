"""Append and attention of several layers captured together, as a decoding step is, and replayed while the sequences
grow: the same bits as the calls made one by one."""
import numpy as np
import pytest
import torch

import diffuse_moe as dm


@pytest.mark.gpu
@pytest.mark.parametrize("kv_type", ["e4m3", "bf16", "f16"])
@pytest.mark.parametrize("rows", [1, 3, 32])
def test_captured_steps_are_the_eager_ones(kv_type, rows):
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    n_layer, n_seq, steps = 3, 3, 6
    caches = [dm.PagedKV(n_pages=40, n_head_kv=2, head_dim=128, page_size=32, kv_type=kv_type, n_layer=n_layer) for _ in "ab"]
    table = torch.from_numpy(np.random.default_rng(1).permutation(39).astype(np.int32).reshape(n_seq, 13)).cuda()
    start = torch.arange(n_seq + 1, dtype=torch.int32, device="cuda") * rows
    w = 1 + 0.1 * torch.randn(128, generator=torch.Generator(device="cuda").manual_seed(0), device="cuda")
    lens = [torch.zeros(n_seq, dtype=torch.int32, device="cuda") for _ in "ab"]
    batches = [kv.batch(table, start, n, rows) for kv, n in zip(caches, lens)]
    x = torch.empty(n_seq * rows, 12 * 128, device="cuda")

    def step(kv, batch):
        h = x
        for il in range(n_layer):
            q = kv.append(il, h, batch, n_head=8, q_norm=w, k_norm=w, rotary_dim=64, q_type=torch.bfloat16)
            o = kv.attend(il, q, batch, block_length=rows)
            h = h + 0.1 * o.float().flatten(1).repeat(1, 2)[:, : 12 * 128]
        return h

    x.zero_(), lens[1].fill_(rows)
    step(caches[1], batches[1])  # warm; every position of it is written again below
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(caches[1], batches[1])
    base = torch.tensor([0, 45, 200], dtype=torch.int32)
    for kv in caches:  # what stands before the first step, the same in both
        g = torch.Generator(device="cuda").manual_seed(3)
        for t in (kv.k, kv.v):
            t.copy_(torch.randn(t.shape, generator=g, device="cuda").to(t.dtype))
        if kv_type == "e4m3":
            kv.k_scale.view(torch.uint8).fill_(126), kv.v_scale.view(torch.uint8).fill_(125)
    g = torch.Generator(device="cuda").manual_seed(2)
    for i in range(steps):
        x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
        for n in lens:
            n.copy_(base + (i + 1) * rows)
        want = step(caches[0], batches[0])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
    for kv in caches:
        kv.check()
    for name in ("k", "v") + (("k_scale", "v_scale") if kv_type == "e4m3" else ()):
        assert torch.equal(*(getattr(kv, name).view(torch.uint8) for kv in caches))

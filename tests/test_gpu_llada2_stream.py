"""forward_paged(stream=...): the whole forward runs there, not the paged cache's calls alone."""
import numpy as np
import pytest
import torch

from test_gpu_llada2_paged import dense_model


@pytest.mark.gpu
def test_forward_paged_on_a_given_stream():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    cfg, model = dense_model()
    tokens = torch.as_tensor(np.random.default_rng(2).integers(0, cfg.n_vocab - 1, size=96), device="cuda")
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    got = []
    for other in (False, True):
        kv = model.new_paged(3, "bf16", page_size=32)
        batch = kv.batch(i32(2, 0, 1)[None], i32(0, 96), i32(96), 96)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        torch.cuda._sleep(200_000_000)  # the current stream is busy for a tenth of a second
        logits = model.forward_paged(tokens, kv, batch, stream=side.cuda_stream if other else None)
        side.synchronize() if other else torch.cuda.synchronize()
        got.append(logits.cpu())
        kv.check()
    assert torch.equal(got[0], got[1])

"""The model over the paged cache on the GPU: forward_paged against forward, and generation."""
import numpy as np
import pytest
import torch

import llada2
from test_gpu_llada2 import rel, tiny_model


@pytest.fixture(autouse=True)
def _need_gpu():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    torch.backends.cuda.matmul.allow_tf32 = False


def dense_model():
    """No MoE blocks: their routing jumps where scores are near, which hides what the cache's rounding does."""
    cfg = llada2.LLaDA2Config(n_layer=3, n_embd=256, n_head=4, n_head_kv=2, head_dim=64, rotary_dim=32, n_ff=512,
                              first_k_dense=3, n_vocab=1000, rope_base=10000.0, mask_token_id=999)
    return cfg, llada2.LLaDA2Model(cfg, llada2.LLaDA2Model.random_weights(cfg, seed=5), {}, dtype=torch.float32)


# Attention's output o comes from rounded q, k, v, weights and output. With normalised queries and keys a score is at
# most about sqrt(head_dim) = 8, so k's (and q's) half steps u move a weight by up to 8 u each, v's and the others by
# u: at most (8 u_k + 8 u_q + u_v + 2 u) of o. o enters the residual (standard deviation 1) through a matrix of gain
# 0.02 * sqrt(256) = 0.32, in 3 blocks: 0.96 of that in the logits. f16: 19 * 2^-11 = 0.0093; bf16: 19 * 2^-8 = 0.074;
# e4m3 (k and v 2^-4, the rest bf16's): 9 * 2^-4 + 10 * 2^-8 = 0.6.
LOGITS = {"f16": 0.0093, "bf16": 0.074, "e4m3": 0.6}


@pytest.mark.gpu
@pytest.mark.parametrize("kv_type", ["f16", "bf16", "e4m3"])
def test_forward_paged_matches_forward(kv_type):
    cfg, model = dense_model()
    rng = np.random.default_rng(2)
    seqs = [torch.as_tensor(rng.integers(0, cfg.n_vocab - 1, size=n), device="cuda") for n in (96, 160)]
    kv = model.new_paged(9, kv_type, page_size=32)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    table = torch.tensor([[7, 2, 5, -1, -1], [0, 8, 1, 3, 4]], dtype=torch.int32, device="cuda")
    model.forward_paged(seqs[0][:64], kv, kv.batch(table[:1].contiguous(), i32(0, 64), i32(64), 64))
    got = model.forward_paged(torch.cat([seqs[0][64:], seqs[1]]), kv, kv.batch(table, i32(0, 32, 192), i32(96, 160), 160))
    kv.check()
    want = torch.cat([model.forward(seqs[0], 0)[64:], model.forward(seqs[1], 0)])
    err = rel(got.cpu().numpy(), want.cpu().numpy())
    assert err <= LOGITS[kv_type], err


@pytest.mark.gpu
@pytest.mark.parametrize("kv_type", ["bf16", "e4m3"])
def test_generation_over_pages(kv_type):
    cfg, w, model, _ = tiny_model()
    rng = np.random.default_rng(3)
    prompts = [rng.integers(0, cfg.n_vocab - 1, size=n) for n in (70, 9, 64)]
    seqs, forwards = llada2.generate_batch(model, prompts, 60, steps=8, threshold=0.95, kv_type=kv_type)
    for p, s in zip(prompts, seqs):
        assert len(s) == -(-(len(p) + 60) // 32) * 32
        assert np.array_equal(s[: len(p)], p) and not np.any(s == cfg.mask_token_id)
    assert 1 <= forwards <= 1 + 8 * 3  # one for the prompts' whole blocks, 8 steps of at most 3 blocks each
    one, n = llada2.generate(model, prompts[1], 60, steps=8, threshold=0.95, kv_type=kv_type)
    assert np.array_equal(one[:9], prompts[1]) and not np.any(one == cfg.mask_token_id) and 1 <= n <= 1 + 8 * 3

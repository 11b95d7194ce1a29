"""The paged forward and the batched generation loop (diffuse-cpp_b200/llada2.py) on the CPU: the cache's two
kernels are replaced by their float64 restatement (kv_ref.py) over float32 pages, the MoE layers and the sampler
by the oracle. A batch of prompts of unequal length commits the tokens that each prompt alone does when the
whole window is recomputed at every step."""
import numpy as np
import pytest
import torch

import kv_ref
import llada2
from test_llada2_cpu import cpu_model, oracle_sampler


class Batch:
    def __init__(self, page_table, q_start, kv_len, max_q_len):
        self.table, self.start, self.lens = page_table.numpy(), q_start.numpy(), kv_len.numpy()
        assert page_table.dtype == q_start.dtype == kv_len.dtype == torch.int32
        assert max_q_len == np.diff(self.start).max()


class Pages:
    """PagedKV's contract in float32 pages, by the restatement."""

    kv_type = "bf16"

    def __init__(self, cfg, n_pages, page_size):
        self.cfg, self.n_pages, self.page_size = cfg, n_pages, page_size
        self.k, self.v = (np.full((cfg.n_layer, n_pages * page_size, cfg.n_head_kv, cfg.head_dim), np.nan) for _ in "kv")
        self.batch = Batch

    def slots(self, batch, i, lo, hi):
        p = np.arange(lo, hi)
        pages = batch.table[i, p // self.page_size]
        assert (pages >= 0).all()
        return pages * self.page_size + p % self.page_size

    def append(self, il, qkv, batch, n_head, q_norm, k_norm, eps, rotary_dim, rope_base, q_type, stream):
        c, n = self.cfg, qkv.shape[0]
        assert n == batch.start[-1]
        x = qkv.numpy().astype(np.float64).reshape(n, n_head + 2 * c.n_head_kv, c.head_dim)
        out = np.empty((n, n_head, c.head_dim))
        for i, (a, b) in enumerate(zip(batch.start[:-1], batch.start[1:])):
            pos = np.arange(batch.lens[i] - (b - a), batch.lens[i])
            rot = lambda y, w: kv_ref.norm_rotate(y, w.numpy(), pos, rotary_dim, rope_base, eps)  # noqa: E731
            out[a:b] = rot(x[a:b, :n_head], q_norm)
            at = self.slots(batch, i, pos[0], batch.lens[i])
            self.k[il, at] = rot(x[a:b, n_head:n_head + c.n_head_kv], k_norm)
            self.v[il, at] = x[a:b, n_head + c.n_head_kv:]
        return torch.from_numpy(out)

    def attend(self, il, q, batch, block_length, stream):
        c = self.cfg
        out = np.empty(q.shape)
        for i, (a, b) in enumerate(zip(batch.start[:-1], batch.start[1:])):
            at = self.slots(batch, i, 0, batch.lens[i])
            for r in range(a, b):
                see = at[: (batch.lens[i] - (b - r)) // block_length * block_length + block_length]
                for h in range(c.n_head):
                    g = h // (c.n_head // c.n_head_kv)
                    out[r, h] = kv_ref.attend_row(q[r, h].numpy(), self.k[il, see, g], self.v[il, see, g], c.head_dim ** -0.5,
                                                  np.ones(len(see)))[0]
        return torch.from_numpy(out.astype(np.float32))


def test_paged_forward_is_the_forward():
    cfg, w, model, _ = cpu_model()
    rng = np.random.default_rng(4)
    seqs = [torch.as_tensor(rng.integers(0, cfg.n_vocab - 1, size=n)) for n in (96, 64)]
    kv = Pages(cfg, 9, 32)
    table = torch.tensor([[7, 2, 5], [0, 8, -1]], dtype=torch.int32)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    # sequence 0's first two blocks, then its last one beside all of sequence 1
    model.forward_paged(seqs[0][:64], kv, kv.batch(table[:1], i32(0, 64), i32(64), 64))
    got = model.forward_paged(torch.cat([seqs[0][64:], seqs[1]]), kv, kv.batch(table, i32(0, 32, 96), i32(96, 64), 64)).numpy()
    want = torch.cat([model.forward(seqs[0], 0)[64:], model.forward(seqs[1], 0)]).numpy()
    assert np.linalg.norm(got - want) / np.linalg.norm(want) <= 1e-5


def test_batched_generation_is_each_prompts_own():
    cfg, w, model, _ = cpu_model()
    w["output"][cfg.mask_token_id] = 0.0
    model.w["output"][cfg.mask_token_id] = 0.0
    rng = np.random.default_rng(3)
    prompts = [rng.integers(0, cfg.n_vocab - 1, size=n) for n in (70, 5, 64)]
    kv = Pages(cfg, 8, 64)
    got, forwards = llada2.generate_batch(model, prompts, 30, steps=4, threshold=0.95, kv=kv, sampler=oracle_sampler)
    most = 0
    for p, s in zip(prompts, got):
        alone, n = llada2.generate(model, p, 30, steps=4, threshold=0.95, use_cache=False, sampler=oracle_sampler)
        assert np.array_equal(s, alone)
        most = max(most, n)
    assert forwards <= most + 1  # the prompts' whole blocks, then every step of the longest


def test_batched_generation_checks():
    cfg, w, model, _ = cpu_model()
    with pytest.raises(ValueError, match="need 4 pages"):
        llada2.generate_batch(model, [np.arange(70)], 40, kv=Pages(cfg, 3, 32), sampler=oracle_sampler)
    with pytest.raises(ValueError, match="paged cache"):
        llada2.generate(model, np.arange(8), 4, kv_type="bf16", use_cache=False)
    seqs, forwards = llada2.generate_batch(model, [], 40, kv=Pages(cfg, 3, 32), sampler=oracle_sampler)
    assert seqs == [] and forwards == 0

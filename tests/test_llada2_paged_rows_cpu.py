"""The paged forward's output projection runs on the rows whose logits are read: none of a prefill's, the last block
of each sequence in a denoising step. Long prefills are cut into calls of a bounded number of rows."""
import numpy as np
import pytest
import torch

import llada2
from test_llada2_cpu import cpu_model, oracle_sampler
from test_llada2_paged_cpu import Pages


def projected(model, monkeypatch):
    """Rows of every output projection from now on."""
    rows, lin = [], model._lin

    def spy(x, name):
        if name == "output":
            rows.append(x.shape[0])
        return lin(x, name)

    monkeypatch.setattr(model, "_lin", spy)
    return rows


def test_logits_of_chosen_rows(monkeypatch):
    cfg, w, model, _ = cpu_model()
    tokens = torch.as_tensor(np.random.default_rng(4).integers(0, cfg.n_vocab - 1, size=96))
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    rows = projected(model, monkeypatch)
    got = []
    for which in (None, torch.tensor([95, 3, 64]), torch.tensor([], dtype=torch.int64)):
        kv = Pages(cfg, 3, 32)
        got.append(model.forward_paged(tokens, kv, kv.batch(table, i32(0, 96), i32(96), 96), rows=which))
        assert np.isfinite(kv.k).all()  # the keys are written all the same
    assert torch.allclose(got[1], got[0][[95, 3, 64]], rtol=1e-5, atol=1e-5)
    assert got[2].shape == (0, cfg.n_vocab)
    assert sum(rows) == 96 + 3


@pytest.mark.parametrize("prefill_rows", [None, 32, 96])
def test_generation_projects_what_it_samples(monkeypatch, prefill_rows):
    cfg, w, model, _ = cpu_model()
    w["output"][cfg.mask_token_id] = 0.0
    model.w["output"][cfg.mask_token_id] = 0.0
    if prefill_rows is not None:
        monkeypatch.setattr(llada2, "PREFILL_ROWS", prefill_rows)
    prompts = [np.random.default_rng(3).integers(0, cfg.n_vocab - 1, size=n) for n in (200, 5, 130, 40)]
    rows, calls, forward = projected(model, monkeypatch), [], model.forward_paged
    monkeypatch.setattr(model, "forward_paged", lambda tokens, *a, **k: (calls.append(len(tokens)), forward(tokens, *a, **k))[1])
    kv = Pages(cfg, 14, 64)
    got, forwards = llada2.generate_batch(model, prompts, 30, steps=4, threshold=0.95, kv=kv, sampler=oracle_sampler)
    assert forwards == len(calls)
    prefill = 160 + 96  # the whole blocks but the last of 200 and 130
    if prefill_rows is not None:
        done = np.cumsum(calls)
        n = int(np.searchsorted(done, prefill)) + 1
        assert done[n - 1] == prefill and max(calls[:n]) <= prefill_rows
    else:
        assert calls[0] == prefill
    assert max(rows) <= 32 * len(prompts)
    for p, s in zip(prompts, got):
        alone, _ = llada2.generate(model, p, 30, steps=4, threshold=0.95, use_cache=False, sampler=oracle_sampler)
        assert np.array_equal(s, alone)

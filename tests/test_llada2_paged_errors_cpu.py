"""What the paged cache's kernels report ends a generation: tokens from attention that is not complete, or that read
wrong pages, are not returned."""
import numpy as np
import pytest

import diffuse_moe as dm
import llada2
from test_llada2_cpu import cpu_model, oracle_sampler
from test_llada2_paged_cpu import Pages


class Reporting(Pages):
    """Pages with an error word that the n-th attention sets."""

    def __init__(self, cfg, n_pages, page_size, at):
        super().__init__(cfg, n_pages, page_size)
        self.at, self.calls, self.bits = at, 0, 0

    def attend(self, *a, **k):
        self.calls += 1
        if self.calls == self.at:
            self.bits = 4
        return super().attend(*a, **k)

    def check(self, all_streams=True):
        if self.bits:
            self.bits = 0
            raise dm.DmoeError(6, "paged cache: a device-side wait timed out")


@pytest.mark.parametrize("at", ["prefill", "first", "last"])
def test_reports_end_a_generation(at):
    cfg, w, model, _ = cpu_model()
    w["output"][cfg.mask_token_id] = 0.0
    model.w["output"][cfg.mask_token_id] = 0.0
    prompt = np.random.default_rng(3).integers(0, cfg.n_vocab - 1, size=70)
    kv = Reporting(cfg, 8, 64, 0)
    _, forwards = llada2.generate_batch(model, [prompt], 20, steps=4, threshold=0.95, kv=kv, sampler=oracle_sampler)
    assert kv.calls == forwards * cfg.n_layer
    kv = Reporting(cfg, 8, 64, {"prefill": 1, "first": cfg.n_layer + 1, "last": forwards * cfg.n_layer}[at])
    with pytest.raises(dm.DmoeError, match="timed out"):
        llada2.generate_batch(model, [prompt], 20, steps=4, threshold=0.95, kv=kv, sampler=oracle_sampler)
    assert kv.bits == 0
    if at != "last":  # found at the next step, not at the end
        assert kv.calls <= 2 * cfg.n_layer


def test_a_prefill_alone_is_checked():
    cfg, w, model, _ = cpu_model()
    prompt = np.random.default_rng(3).integers(0, cfg.n_vocab - 1, size=64)
    kv = Reporting(cfg, 8, 64, 1)
    with pytest.raises(dm.DmoeError, match="timed out"):
        llada2.generate_batch(model, [prompt], 0, steps=4, kv=kv, sampler=oracle_sampler)

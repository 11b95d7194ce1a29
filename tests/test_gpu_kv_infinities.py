"""Infinite values in 16-bit pages: a row that sees +inf in a column has +inf there, -inf likewise, NaN where it sees
both or a NaN; rows that do not see them, and other columns, are as they were. Whatever the tile they lie in."""
import numpy as np
import pytest
import torch

from test_gpu_kv import Setup, queries

INF = float("inf")


@pytest.fixture(autouse=True)
def _need_gpu():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["bf16", "f16"])
@pytest.mark.parametrize("rows,ctx", [(1, 161), (3, 161), (60, 161), (60, 30), (300, 4000)])
def test_infinite_values_keep_their_sign(kv, rows, ctx):
    s = Setup([rows], [ctx], kv, 8, 2, 128, page=64, seed=8)
    s.ctx = s.lens
    s.fill()
    q = queries(s, "bf16", size=0.3)  # no weight vanishes
    clean = s.kv.attend(0, q, s.batch, block_length=1).double().cpu().numpy()
    # (position, column, value): in a tile that all rows see (where there is one), at the first, a middle and the last row
    last = ctx + rows - 1
    put = [(3, 2, INF), (ctx, 5, INF), (ctx, 40, -INF), (ctx + rows // 2, 9, -INF), (ctx + rows // 2, 77, INF),
           (last, 5, -INF), (last, 77, INF), (ctx + rows // 3, 100, INF), (last, 100, float("nan")), (3, 127, -INF), (last, 127, INF)]
    want = clean.copy()
    for (p, d), x in {(p, d): x for p, d, x in put}.items():  # one row: the last of those for an element stands
        s.kv.v[0, int(s.table[0, p // s.page]), 1, p % s.page, d] = x
        with np.errstate(invalid="ignore"):  # inf - inf
            want[max(0, p - ctx):, 4:, d] += x
    got = s.kv.attend(0, q, s.batch, block_length=1).double().cpu().numpy()
    s.kv.check()
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(np.isposinf(got), np.isposinf(want)) and np.array_equal(np.isneginf(got), np.isneginf(want))
    fin = np.isfinite(want)
    assert np.allclose(got[fin], clean[fin], rtol=2.0 ** -6, atol=1e-3)

"""A position that holds most of the weight, with a value near zero (an attention sink): the rest of the
positions keep their precision on pages whose products are f16."""
import numpy as np
import pytest
import torch

import kv_ref
from test_gpu_kv import Setup


@pytest.fixture(autouse=True)
def _need_gpu():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"


# Weights are held in f16 as multiples of a reference that lies 2^15 (single tokens) or at least 2^7 (tiles) below
# the largest of their running maximum's positions, so half of their smallest step is 2^-25 * 2^-15 or 2^-25 * 2^-7 of it.
def held_to(rows):
    return 2.0 ** -40 if rows <= 4 else 2.0 ** -32


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["e4m3", "f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 4, 64])
@pytest.mark.parametrize("sink,unit", [(20.37, 0), (21.567, 0), (23.4, 0), (24.3, 0), (1.567, 20)])
def test_positions_beside_a_sink(kv, rows, sink, unit):
    """Query rows are the first unit vector, key 0 too, and the other keys have no such element: their weights are all
    2^-sink of the first one's, so that their roundings add up. `unit`: the exponent of the value scale of the sink's
    block, whose other values lie in its lowest codes."""
    if unit and kv != "e4m3":
        pytest.skip("scales belong to 8-bit pages")
    n, n_seq = 16384, 160  # sequences over the same pages: every CTA has whole items, and the sink comes first in each
    s = Setup([rows], [n - rows], kv, 8, 2, 128, page=64, seed=1, fill=False)
    g = torch.Generator(device="cuda").manual_seed(2)
    dtype = s.kv.k.dtype
    for t, low in ((s.kv.k, -1.0), (s.kv.v, 0.25)):  # values of one sign: the output is of their size
        x = low + (1.0 - low) * torch.rand(t.shape, generator=g, device="cuda")
        t.copy_(x.to(dtype))
    if kv == "e4m3":
        for t in (s.kv.k_scale, s.kv.v_scale):
            t.view(torch.uint8).fill_(127)
    s.kv.k.view(torch.uint8 if kv == "e4m3" else dtype)[..., 0] = 0
    first = int(s.table[0, 0])
    s.kv.k[0, first, :, 0] = torch.eye(1, 128, device="cuda").to(dtype)
    s.kv.v.view(torch.uint8 if kv == "e4m3" else dtype)[0, first, :, 0] = 0
    if unit:
        s.kv.v_scale.view(torch.uint8)[0, first, :, 0] = 127 + unit
        s.kv.v.view(torch.uint8)[0, first, :, :32] = 0
    scale = sink * float(np.log(2.0))
    q = torch.zeros(n_seq * rows, 8, 128, device="cuda", dtype=torch.float16)
    q[..., 0] = 1.0
    lse = torch.empty(n_seq * rows, 8, device="cuda")
    i32 = lambda a: torch.from_numpy(np.asarray(a, np.int32)).cuda()  # noqa: E731
    batch = s.kv.batch(i32(np.repeat(s.table, n_seq, 0)), i32(rows * np.arange(n_seq + 1)), i32([n] * n_seq), rows)
    out = s.kv.attend(0, q, batch, block_length=1, scale=scale, lse=lse)
    s.kv.check()
    out, lse = out.view(n_seq, rows, 8, 128)[[0, 31, 80, 159]].double().cpu().numpy(), lse.view(n_seq, rows, 8)[[0, 31, 80, 159]].double().cpu().numpy()
    k, _ = s.held("k", 0, n)
    v, vu = s.held("v", 0, n)
    e0 = np.zeros(128)
    e0[0] = 1.0
    bf = kv == "bf16"
    for r in sorted({0, rows // 2, rows - 1}):
        see = n - rows + r + 1
        for h in (0, 5, 7):
            kk, vv, u = k[:see, h // 4], v[:see, h // 4], vu[:see, h // 4]
            ref, rl, size, step = kv_ref.attend_row(e0, kk, vv, scale, u)
            score = kv_ref.score_error(e0, kk[:1], scale, kv, "f16")
            rel = kv_ref.HALF_STEP["bf16" if bf else "f16"] + 2 * np.expm1(score + 2.0 ** -21) + (see / 8 + 64) * 2.0 ** -23
            tol = rel * size + (0.0 if bf else held_to(rows)) * step + kv_ref.HALF_STEP["f16"] * np.abs(ref) * 1.01 + 2.0 ** -25
            err = np.abs(out[:, r, h] - ref)
            assert (err <= tol).all(), (r, h, float((err / tol).max()), float((err / np.abs(ref)).max()))
            assert (np.abs(lse[:, r, h] - rl) <= score + 2.0 ** -18 + abs(rl) * 2.0 ** -21).all()

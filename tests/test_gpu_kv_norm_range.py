"""QK norm of rows whose squares leave the range of 32 bits: x / sqrt(mean x^2 + eps) is of ordinary size."""
import numpy as np
import pytest
import torch

import diffuse_moe as dm
import kv_ref


@pytest.fixture(autouse=True)
def _need_gpu():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["e4m3", "bf16", "f16"])
@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("size,eps", [(1e18, 1e-6), (1e19, 1e-6), (1e25, 1e-6), (1e37, 1e-6), (1e-3, 0.0), (1e-17, 0.0), (1e-22, 0.0), (1e-30, 0.0)])
@pytest.mark.parametrize("dim,rot", [(128, 64), (64, 0)])
def test_norm_of_any_size(kv, io, size, eps, dim, rot):
    n, nh, nk = 5, 4, 2
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(n, nh + 2 * nk, dim, generator=g, device="cuda")
    x[1] *= 1e-3  # a row of another size beside it
    x[2, 1] *= 1e2 if size > 1 and size < 1e36 else 1.0
    x[:, : nh + nk] *= size
    x[3, : nh + nk] = torch.randn(nh + nk, dim, generator=g, device="cuda")  # and one of ordinary size
    x = x.to(torch.float32 if io == "f32" else torch.bfloat16)
    w = 1 + 0.2 * torch.randn(2, dim, generator=g, device="cuda")
    cache = dm.PagedKV(n_pages=1, n_head_kv=nk, head_dim=dim, page_size=32, kv_type=kv)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    batch = cache.batch(i32([[0]]), i32([0, n]), i32([n]), n)
    q = cache.append(0, x.flatten(1), batch, n_head=nh, q_norm=w[0], k_norm=w[1], eps=eps, rotary_dim=rot, rope_base=1e4,
                     q_type=torch.float32)
    cache.check()
    xn, pos = x.double().cpu().numpy(), np.arange(n)
    # eps as the call has it, in 32 bits
    want = [kv_ref.norm_rotate(xn[:, a:b], w[i].cpu().numpy(), pos, rot, 1e4, float(np.float32(eps)))
            for i, (a, b) in enumerate(((0, nh), (nh, nh + nk)))]
    err = np.abs(q.double().cpu().numpy() - want[0])
    assert (err <= kv_ref.HALF_STEP["f32"] * np.abs(want[0]) + kv_ref.ROTATE_ERR * kv_ref.pair_norm(want[0], rot)).all()
    k = cache.k[0, 0, :, :n].float()
    unit = np.ones((nk, 1, 1))
    if kv == "e4m3":
        unit = 2.0 ** (cache.k_scale.view(torch.uint8)[0, 0].double().cpu().numpy()[:, :, None] - 127)
    k = (k.double().cpu().numpy() * unit).transpose(1, 0, 2)
    slack = kv_ref.ROTATE_ERR * kv_ref.pair_norm(want[1], rot)
    tol = kv_ref.HALF_STEP[kv] * (np.abs(want[1]) + slack) + slack
    tol = tol + (2.0 ** -10 * unit.transpose(1, 0, 2) if kv == "e4m3" else 2.0 ** -25 if kv == "f16" else 0.0)
    assert (np.abs(k - want[1]) <= tol).all()

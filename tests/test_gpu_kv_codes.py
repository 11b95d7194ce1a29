"""Keys of 8-bit pages: every code and scale is that of the exact value, not of one that was rounded on the way. The
inputs are made so that the exact keys lie within a few 2^-25 of the border between two codes, or of a scale's
border, where 32-bit arithmetic (restated here) falls on the wrong side about every other time."""
import numpy as np
import pytest
import torch

import diffuse_moe as dm
import kv_ref

#: Keys closer to a border than this (relative) are left out: the angle's own error in 64 bits, 64 products of
#: 2^-53 each by an angle of at most 4000, and the sums of squares.
NEAR = 64 * 4000 * 2.0 ** -53 * 4


@pytest.fixture(autouse=True)
def _need_gpu():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"


def keys_of(qkv, n, n_ctx, dim, norm, rot, base, eps=1e-6):
    """The appended codes [n, dim] and scale exponents [n / 32] of one key head."""
    kv = dm.PagedKV(n_pages=(n_ctx + n) // 32, n_head_kv=1, head_dim=dim, page_size=32, kv_type="e4m3")
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    table = torch.arange(kv.n_pages, dtype=torch.int32, device="cuda")[None]
    kv.append(0, qkv, kv.batch(table, i32([0, n]), i32([n_ctx + n]), n), n_head=1, k_norm=norm, eps=eps, rotary_dim=rot,
              rope_base=base, q_type=torch.bfloat16)
    kv.check()
    first = n_ctx // 32
    return (kv.k.view(torch.uint8)[0, first:, 0].reshape(n, dim).cpu().numpy(),
            kv.k_scale.view(torch.uint8)[0, first:, 0, 0].cpu().numpy().astype(int) - 127)


def rotated_near_ties(dim, rot, n_ctx):
    """Inputs [768, 3, dim] whose key is, after the rotation, next to a tie in half of the rotated elements; in
    every other block the largest element is next to the border of a scale. The exact keys, and by 32-bit arithmetic."""
    n, base, h = 768, 10000.0, rot // 2
    rng = np.random.default_rng(dim + rot)
    pos = n_ctx + np.arange(n)
    ang = pos[:, None] * base ** (-2.0 * np.arange(h) / rot)[None, :]
    c, s = np.cos(ang), np.sin(ang)
    mid = (kv_ref.POSITIVE[1:127] + kv_ref.POSITIVE[:126]) / 2
    x = np.zeros((n, 3, dim), np.float32)
    for b in range(0, n, 32):
        at, border = slice(b, b + 32), b % 64 == 0
        t = rng.choice(mid[(mid > 1) & (mid < (100 if border else 200))], (32, h)) * rng.choice([-1, 1], (32, h))
        second = rng.uniform(-20, 20, (32, h)).astype(np.float32)
        ok = np.abs(c[at]) > 0.5  # x1 cos - x2 sin = t, solved for x1
        x[at, 1, :h] = np.where(ok, (t + second * s[at]) / np.where(ok, c[at], 1.0), 0.0)
        x[at, 1, h:rot] = second
        x[at, 1, rot:] = rng.uniform(-100, 100, (32, dim - rot))
        if border:
            r = b + int(np.argmax(np.abs(c[at, 1])))
            x[r, 1, 1] = (448.0 + np.float64(x[r, 1, h + 1]) * s[r, 1]) / c[r, 1]
    exact = kv_ref.norm_rotate(x[:, 1:2].astype(np.float64), None, pos, rot, base, 0.0)[:, 0]
    c32, s32, x1, x2 = c.astype(np.float32), s.astype(np.float32), x[:, 1, :h], x[:, 1, h:rot]
    return x, exact, np.concatenate([x1 * c32 - x2 * s32, x2 * c32 + x1 * s32, x[:, 1, rot:]], 1)


@pytest.mark.gpu
@pytest.mark.parametrize("dim,rot", [(128, 64), (128, 128), (64, 32)])
@pytest.mark.parametrize("n_ctx", [0, 3200])
def test_rotated_keys_near_a_tie(dim, rot, n_ctx):
    x, exact, low = rotated_near_ties(dim, rot, n_ctx)
    codes, exps = keys_of(torch.from_numpy(x.reshape(len(x), -1)).cuda(), len(x), n_ctx, dim, None, rot, 10000.0)
    assert check(codes, exps, exact, low) >= 1  # scales that 32-bit arithmetic gets wrong


def check(codes, exps, exact, low):
    """Codes and exponents against the exact keys; `low`, the same keys by 32-bit arithmetic, must differ."""
    mid = (kv_ref.POSITIVE[1:127] + kv_ref.POSITIVE[:126]) / 2
    wrong_scale = wrong_code = tested = 0
    for i, e in enumerate(exps):
        y, z = exact[32 * i:32 * i + 32], low[32 * i:32 * i + 32].astype(np.float64)
        amax = np.abs(y).max()
        border = 448.0 * 2.0 ** np.round(np.log2(amax / 448.0))
        if abs(amax / border - 1) > NEAR:
            assert e == kv_ref.exponent(amax), (i, amax)
        wrong_scale += kv_ref.exponent(np.abs(z).max()) != kv_ref.exponent(amax)
        u = 2.0 ** int(e)
        v = np.abs(y) / u
        at = np.searchsorted(mid, v)
        gap = np.minimum(np.abs(v - mid[np.minimum(at, 125)]), np.abs(v - mid[np.maximum(at - 1, 0)]))
        sure = gap > NEAR * np.maximum(v, np.abs(z) / u)
        want = kv_ref.encode(np.clip(y / u, -448, 448))
        assert np.array_equal(codes[32 * i:32 * i + 32][sure], want[sure]), (i, int((codes[32 * i:32 * i + 32] != want)[sure].sum()))
        wrong_code += int((kv_ref.encode(np.clip(z / u, -448, 448)) != want)[sure].sum())
        tested += int(sure.sum())
    assert tested > 0.9 * codes.size
    assert wrong_code >= 20, wrong_code  # 32-bit arithmetic is seen to fail
    return wrong_scale


def normalised_near_ties(rng, dim):
    """A key row and weights that put every normalised element next to a tie."""
    mid = (kv_ref.POSITIVE[1:127] + kv_ref.POSITIVE[:126]) / 2
    x = rng.standard_normal((1, 3, dim)).astype(np.float32) * 3
    x[0, 1, np.abs(x[0, 1]) < 0.1] = 0.7
    xd = x[0, 1].astype(np.float64)
    r = 1 / np.sqrt(np.mean(xd * xd) + float(np.float32(1e-6)))
    t = rng.choice(mid[(mid > 1) & (mid < 200)], dim)
    t[0] = 401.0
    w = (t / (xd * r)).astype(np.float32)
    r32 = np.float32(1) / np.sqrt(np.mean(x[0, 1] * x[0, 1], dtype=np.float32) + np.float32(1e-6))
    return x, w, xd * r * w.astype(np.float64), x[0, 1] * r32 * w


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
def test_normalised_keys_near_a_tie(dim):
    rng = np.random.default_rng(dim)
    codes, exps, exact, low = [], [], [], []
    for _ in range(24):
        x, w, y, z = normalised_near_ties(rng, dim)
        c, e = keys_of(torch.from_numpy(x.reshape(1, -1)).cuda().repeat(32, 1), 32, 0, dim, torch.from_numpy(w).cuda(), 0, 1e4)
        codes.append(c), exps.append(e)
        exact.append(np.repeat(y[None], 32, 0)), low.append(np.repeat(z[None], 32, 0))
    check(np.concatenate(codes), np.concatenate(exps), np.concatenate(exact), np.concatenate(low))

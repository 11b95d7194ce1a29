"""float64 restatement of the paged key/value cache's two operators, for checking dmoe_kv_append and
dmoe_kv_attention (plain numpy; the product never imports it), and the error bounds that the tests hold
the kernels to."""
import numpy as np

BLOCK, E_MIN, E_MAX = 32, -60, 120
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8, "e4m3": 2.0 ** -4}

# the values of the e4m3 codes: sign, 4 exponent bits (bias 7), 3 mantissa bits, 0x7f = NaN
_c = np.arange(128)
POSITIVE = np.where(_c < 8, _c * 2.0 ** -9, (8 + _c % 8) * 2.0 ** (_c // 8 - 10.0))
POSITIVE[127] = np.nan
DECODE = np.concatenate([POSITIVE, -POSITIVE])


def encode(x):
    """Nearest e4m3 code, ties to the even mantissa; |x| <= 448 where finite, NaN otherwise."""
    a = np.abs(x)
    fin = np.isfinite(a)
    assert np.all(a[fin] <= 448)
    table = POSITIVE[:127]
    mid = (table[1:] + table[:-1]) / 2
    a0 = np.where(fin, a, 0.0)
    lo = np.searchsorted(mid, a0, side="left")   # the lower code at a tie
    tie = (lo < 126) & (a0 == mid[np.minimum(lo, 125)])
    code = np.where(tie & (lo % 2 == 1), lo + 1, lo)
    code = np.where(fin, code, 127)
    return (code + 128 * np.signbit(x)).astype(np.uint8)


def exponent(amax):
    e = E_MIN
    while e < E_MAX and amax > 448.0 * 2.0 ** e:
        e += 1
    return e


def norm_rotate(x, w, pos, rotary_dim, base, eps):
    """x [n, heads, d] -> normalised (w not None) and rotated at positions pos [n]."""
    x = x.astype(np.float64)
    if w is not None:
        x = x / np.sqrt(np.mean(x * x, axis=-1, keepdims=True) + eps) * w.astype(np.float64)
    h = rotary_dim // 2
    ang = pos[:, None] * np.array([base ** (-2.0 * i / rotary_dim) for i in range(h)])[None, :]
    z = (x[..., :h] + 1j * x[..., h:2 * h]) * np.exp(1j * ang)[:, None, :]
    return np.concatenate([z.real, z.imag, x[..., 2 * h:]], axis=-1)


def pair_norm(x, rotary_dim):
    """The size that rounding errors of a rotated element are relative to: its pair's norm."""
    h = rotary_dim // 2
    n = np.abs(x[..., :h] + 1j * x[..., h:2 * h])
    return np.concatenate([n, n, np.abs(x[..., 2 * h:])], axis=-1)


#: 32-bit arithmetic of norm and rotation, relative to pair_norm: the sum of squares (8 fused additions and
#: 4 shuffles: 12 half steps, halved by the root), root, division, two products (4), the rotation (3 each
#: side of a sum that may be twice the result: 6), sincospif (2 steps = 4), the fraction of the turn rounded
#: to 24 bits (2 pi 2^-26 = 1.6 half steps): under 24; doubled.
ROTATE_ERR = 48 * 2.0 ** -24


def attend_row(q, k, v, scale, unit):
    """softmax(scale k q) v over the given positions: o, the logarithm of the sum, and what errors are
    relative to: sum w |v| / sum w, and max_j (w_j unit_j) sum_j |v_j| / unit_j / sum w (the size of the
    smallest step of the rounded weights). Zeros where there are no positions."""
    d = v.shape[1]
    if len(k) == 0:
        return np.zeros(d), -np.inf, np.zeros(d), np.zeros(d)
    s = (k @ q) * scale
    m = s.max()
    w = np.exp(s - m)
    t = w.sum()
    return (w @ v) / t, m + np.log(t), (w @ np.abs(v)) / t, (w * unit).max() / t * (np.abs(v) / unit[:, None]).sum(0)


def score_error(q, k, scale, kv, io):
    """Bound of a score's error: 32-bit sums of head_dim + 16 additions that may truncate (a whole step,
    2^-23, each), the factor's and the exponent's rounding (2^-21); a query element rounded to the products'
    type where that is not exact: f16 queries on bf16 pages, or below 2^-14 of the row's largest."""
    dot = scale * np.max(np.abs(k) @ np.abs(q))
    rounding = HALF_STEP["bf16"] if kv == "bf16" and io == "f16" else 0.0
    small = scale * 2.0 ** -25 * np.max(np.abs(q)) * 2 * np.max(np.abs(k).sum(1)) if kv != "bf16" else 0.0
    return dot * ((len(q) + 16) * 2.0 ** -23 + 2.0 ** -21 + rounding) + small


def attend_tolerance(o, a, step, q, k, scale, kv, io):
    """Bound of |kernel - o|: weights rounded once to the products' type (bf16 on bf16 pages, else f16, whose
    smallest half step is 2^-25); the scores' errors, in numerator and denominator, and the
    exponentials' (2^-21 each); sums over the positions, 16 a product, that may truncate; the output's half
    step (f16: 2^-25 at least)."""
    if len(k) == 0:
        return np.zeros_like(o)
    bf = kv == "bf16"
    rel = HALF_STEP["bf16" if bf else "f16"] + 2 * np.expm1(score_error(q, k, scale, kv, io) + 2.0 ** -21)
    rel = rel + (len(k) / 8 + 64) * 2.0 ** -23
    return rel * a + (0.0 if bf else 2.0 ** -25) * step + HALF_STEP[io] * np.abs(o) * 1.01 + 2.0 ** -25

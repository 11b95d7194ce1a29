"""The paged key/value cache on the GPU (PagedKV.append, PagedKV.attend) against the float64 restatement
in kv_ref.py: every page type, head layout and row type, lengths from one position on, pages that end
inside a tile, left padding, empty sequences, rows behind the last sequence, strides and alignment, a graph
replayed with longer sequences, another stream, values that are not finite, bad pages and batches."""
import numpy as np
import pytest
import torch

import diffuse_moe as dm
import kv_ref

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6


@pytest.fixture(autouse=True)
def _need_gpu(request):
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"


class Setup:
    """Sequences with `ctx` positions in the cache and `q_lens` new rows each, on shuffled pages."""

    def __init__(self, q_lens, ctx, kv="e4m3", heads=8, heads_kv=2, dim=128, page=64, seed=0, spare_rows=0, fill=True):
        self.rng = np.random.default_rng(seed)
        self.q_lens, self.ctx, self.kv_name = list(q_lens), list(ctx), kv
        self.nh, self.nk, self.d, self.page = heads, heads_kv, dim, page
        self.n = sum(q_lens)
        self.rows = self.n + spare_rows
        self.lens = [a + c for a, c in zip(q_lens, ctx)]
        need = [max(0, -(-x // page)) for x in self.lens]
        self.n_pages = sum(need) + 2
        order = self.rng.permutation(self.n_pages).astype(np.int32)
        self.table = np.full((len(q_lens), max(need + [1])), -7, np.int32)
        at = 0
        for i, m in enumerate(need):
            self.table[i, :m] = order[at:at + m]
            at += m
        self.kv = dm.PagedKV(n_pages=self.n_pages, n_head_kv=heads_kv, head_dim=dim, page_size=page, kv_type=kv)
        self.start = np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32)
        self.batch = self.make_batch(self.lens)
        # unread memory is NaN: what a kernel takes from it shows
        for t in (self.kv.k, self.kv.v):
            t.view(torch.uint8).fill_(0x7f) if kv == "e4m3" else t.fill_(float("nan"))
        if fill:
            self.fill()

    def make_batch(self, lens, max_q_len=None):
        c = lambda a: torch.from_numpy(np.asarray(a, np.int32)).cuda()  # noqa: E731
        return dm.KVBatch(c(self.table), c(self.start), c(lens), max(self.q_lens) if max_q_len is None else max_q_len)

    def fill(self):
        """The positions before the new rows: keys with unequal channels, values of unequal size."""
        g = torch.Generator(device="cuda").manual_seed(int(self.rng.integers(1 << 30)))
        for i, c in enumerate(self.ctx):
            for p0 in range(0, max(c, 0), 32):
                m, pg, of = min(32, c - p0), int(self.table[i, p0 // self.page]), p0 % self.page
                for held, scale in ((self.kv.k, self.kv.k_scale), (self.kv.v, self.kv.v_scale)):
                    x = torch.randn(self.nk, m, self.d, generator=g, device="cuda")
                    x *= torch.exp(0.7 * torch.randn(self.nk, 1, 1, generator=g, device="cuda"))
                    if self.kv_name == "e4m3":
                        e = torch.tensor([kv_ref.exponent(float(a)) for a in x.abs().amax((1, 2)).cpu()], device="cuda")
                        held.view(torch.uint8)[0, pg, :, of:of + m] = torch.ldexp(x, -e[:, None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
                        scale.view(torch.uint8)[0, pg, :, of // 32] = (e + 127).to(torch.uint8)
                    else:
                        held[0, pg, :, of:of + m] = x.to(held.dtype)

    def held(self, which, i, n):
        """float64 [n, heads_kv, d] of sequence i's first n positions, and each one's scale [n, heads_kv]."""
        t = getattr(self.kv, which)[0]
        p = np.arange(n)
        pg = torch.from_numpy(self.table[i, p // self.page].astype(np.int64)).cuda()
        of = torch.from_numpy(p % self.page).cuda()
        if self.kv_name != "e4m3":
            return t[pg, :, of].double().cpu().numpy(), np.ones((n, self.nk))
        x = kv_ref.DECODE[t.view(torch.uint8)[pg, :, of].cpu().numpy()]
        s = getattr(self.kv, which + "_scale")[0].view(torch.uint8)[pg, :, of // 32].cpu().numpy()
        unit = 2.0 ** (s.astype(np.float64) - 127)
        return x * unit[..., None], unit


def queries(s, io, seed=5, size=1.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (size * torch.randn(s.rows, s.nh, s.d, generator=g, device="cuda")).to(TORCH[io])


def check_attend(s, q, io, block, scale=None, out=None, lse=None, batch=None, lens=None, rows=None):
    out = torch.full_like(q, 7.0) if out is None else out
    lse = torch.full(q.shape[:2], 7.0, device="cuda") if lse is None else lse
    got = s.kv.attend(0, q, batch or s.batch, block_length=block, scale=scale, out=out, lse=lse)
    assert got is out
    s.kv.check()
    verify_attend(s, q, io, block, out, lse, scale, lens, rows)


def verify_attend(s, q, io, block, out, lse, scale=None, lens=None, rows=None):
    scale = s.d ** -0.5 if scale is None else scale
    o, ls, qn = out.double().cpu().numpy(), lse.double().cpu().numpy(), q.double().cpu().numpy()
    group = s.nh // s.nk
    for i, (a, n) in enumerate(zip(s.q_lens, s.lens if lens is None else lens)):
        if a == 0:
            continue
        k, ku = s.held("k", i, n)
        v, vu = s.held("v", i, n)
        picks = range(a) if rows is None or a <= rows else sorted({0, a - 1, *s.rng.integers(0, a, rows).tolist()})
        for r in picks:
            pos = n - a + r
            see = min(n, (pos // block + 1) * block) if pos >= 0 else 0
            for h in range(s.nh):
                kk, vv, unit = k[:see, h // group], v[:see, h // group], vu[:see, h // group]
                x = qn[s.start[i] + r, h]
                ref, rl, absolute, step = kv_ref.attend_row(x, kk, vv, scale, unit)
                tol = kv_ref.attend_tolerance(ref, absolute, step, x, kk, scale, s.kv_name, io)
                err = np.abs(o[s.start[i] + r, h] - ref)
                assert (err <= tol).all(), (i, r, h, float((err - tol).max()), float((err / np.maximum(tol, 1e-300)).max()))
                if see == 0:
                    assert ls[s.start[i] + r, h] == -np.inf
                else:
                    lt = kv_ref.score_error(x, kk, scale, s.kv_name, io) + 2.0 ** -18 + abs(rl) * 2.0 ** -21
                    assert abs(ls[s.start[i] + r, h] - rl) <= lt, (i, r, h, ls[s.start[i] + r, h], rl)
    assert bool((out[s.n:] == 7.0).all()) and bool((lse[s.n:] == 7.0).all())


LAYOUTS = [(8, 2, 128), (4, 2, 64), (4, 4, 128), (24, 8, 64), (32, 4, 128), (5, 1, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["e4m3", "bf16", "f16"])
@pytest.mark.parametrize("heads,heads_kv,dim", LAYOUTS)
def test_attend_single_tokens(kv, heads, heads_kv, dim):
    s = Setup([1] * 6, [0, 1, 31, 32, 200, 1030], kv, heads, heads_kv, dim, page=32, seed=heads)
    s.ctx = [c + 1 for c in s.ctx]  # the cache holds every position
    s.fill()
    check_attend(s, queries(s, "bf16"), "bf16", 1)


@pytest.mark.gpu
@pytest.mark.parametrize("kv,io", [("e4m3", "bf16"), ("e4m3", "f16"), ("bf16", "bf16"), ("bf16", "f16"), ("f16", "f16"), ("f16", "bf16")])
@pytest.mark.parametrize("block", [1, 32])
@pytest.mark.parametrize("heads,heads_kv,dim", [(8, 2, 128), (4, 2, 64), (3, 3, 128)])
def test_attend_several_rows(kv, io, block, heads, heads_kv, dim):
    s = Setup([2, 5, 33, 64, 150], [0, 27, 95, 32, 333], kv, heads, heads_kv, dim, page=96, seed=block + heads, spare_rows=3)
    s.ctx = s.lens
    s.fill()
    check_attend(s, queries(s, io), io, block, rows=12)


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["e4m3", "bf16"])
@pytest.mark.parametrize("block", [1, 7, 64, 1 << 20])
def test_attend_block_lengths(kv, block):
    s = Setup([70, 300], [0, 129], kv, 8, 1, 128, page=64, seed=block)
    s.ctx = s.lens
    s.fill()
    check_attend(s, queries(s, "bf16"), "bf16", block, rows=24)


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["e4m3", "bf16", "f16"])
def test_attend_long_and_odd(kv):
    s = Setup([1, 1, 1], [20011, 7, 5555], kv, 8, 2, 128, page=64, seed=3)
    s.ctx = s.lens
    s.fill()
    check_attend(s, queries(s, "bf16"), "bf16", 1)
    s = Setup([17, 40], [9001, 3], kv, 8, 2, 128, page=128, seed=4)
    s.ctx = s.lens
    s.fill()
    check_attend(s, queries(s, "bf16"), "bf16", 32, rows=6)


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["e4m3", "bf16"])
@pytest.mark.parametrize("q_lens", [[1, 2, 2, 0, 1], [40, 5, 100, 0, 33]])
def test_attend_padding_and_empty(kv, q_lens):
    """Left padding (fewer positions than rows), sequences with no rows, with no positions, spare rows."""
    s = Setup(q_lens, [0] * 5, kv, 8, 2, 64, page=32, seed=9, spare_rows=4)
    s.ctx = s.lens
    s.fill()
    lens = [1, 1, 0, 0, 1] if q_lens[0] == 1 else [3, 0, 99, 0, 33]
    check_attend(s, queries(s, "bf16"), "bf16", 1, batch=s.make_batch(lens), lens=lens)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 50])
def test_attend_strides_and_scale(rows):
    s = Setup([rows, rows], [100, 7], "e4m3", 8, 2, 128, seed=2)
    s.ctx = s.lens
    s.fill()
    wide = torch.randn(s.rows, 8 * 128 + 24, device="cuda").to(torch.bfloat16)
    for at, width in ((8, 8 * 128 + 24), (1, 8 * 128 + 24)):  # aligned rows, and rows that start at an odd element
        q = wide[:, at:at + 1024].unflatten(1, (8, 128))
        buf = torch.full((s.rows, width), 7.0, device="cuda", dtype=torch.bfloat16)
        out = buf[:, at:at + 1024].unflatten(1, (8, 128))
        check_attend(s, q, "bf16", 1, scale=0.3, out=out, rows=8)
        assert bool((buf[:, :at] == 7.0).all()) and bool((buf[:, at + 1024:] == 7.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("kv", ["e4m3", "f16"])
def test_attend_extreme_sizes(kv, rows):
    """Values whose sizes differ by far more than 16 bits hold between blocks, one key that takes all the
    weight, and large queries."""
    s = Setup([rows], [300], kv, 4, 2, 128, seed=8)
    s.ctx = s.lens
    s.fill()
    if kv == "e4m3":
        pg = torch.from_numpy(s.table[0].astype(np.int64)).cuda()
        sc = s.kv.v_scale.view(torch.uint8)
        sc[0, pg[0], :, 0] = 127 - 40
        sc[0, pg[1], :, 1] = 127 + 30
        sc[0, pg[2], 0, 0] = 127 - 60
        s.kv.v.view(torch.uint8)[0, pg[3], :, 0:32] = 0  # a block of zeros
        sc[0, pg[3], :, 0] = 127 - 60
    check_attend(s, queries(s, "bf16", size=1.0), "bf16", 1, rows=10)
    check_attend(s, queries(s, "bf16", size=30.0), "bf16", 1, rows=10)
    if kv == "e4m3":
        check_attend(s, queries(s, "bf16", size=1e-30), "bf16", 1, rows=10)


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["e4m3", "bf16", "f16"])
@pytest.mark.parametrize("rows,heads", [(1, 8), (2, 8), (5, 4), (60, 8)])
def test_attend_not_finite_reaches_only_rows_that_see_it(kv, rows, heads):
    s = Setup([rows], [161], kv, heads, 2, 128, seed=8)
    s.ctx = s.lens
    s.fill()
    q = queries(s, "bf16")
    clean = s.kv.attend(0, q, s.batch, block_length=1).clone()
    for r in {rows - 1, rows // 2}:
        keep = {n: getattr(s.kv, n).clone() for n in "kv"}
        for which, d in (("v", 5), ("k", 9)):
            p = 161 + r
            pg = int(s.table[0, p // s.page])
            t = getattr(s.kv, which)
            if kv == "e4m3":
                t.view(torch.uint8)[0, pg, 1, p % s.page, d] = 0x7f
            else:
                t[0, pg, 1, p % s.page, d] = float("nan")
            got = s.kv.attend(0, q, s.batch, block_length=1)
            bad = torch.isnan(got)
            assert not bad[:r].any() and not bad[:, : heads // 2].any()
            if which == "v":
                assert bool(bad[r:, heads // 2:, d].all()) and int(bad.sum()) == (rows - r) * (heads // 2)
            else:
                assert bool(bad[r:, heads // 2:].all())
            ok = ~bad
            assert torch.allclose(got[ok].float(), clean[ok].float(), rtol=2.0 ** -6, atol=1e-3)
            getattr(s.kv, which).copy_(keep[which])


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 40])
def test_attend_graph_stream_and_repeat(rows):
    """Captured once, replayed as the sequences grow; on another stream; bit-equal when repeated."""
    s = Setup([rows, rows], [900, 2500], "e4m3", 8, 2, 128, seed=6)
    s.ctx = s.lens
    s.fill()
    q = queries(s, "bf16")
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device="cuda")
    first = s.kv.attend(0, q, s.batch, block_length=32).clone()
    for _ in range(3):
        assert torch.equal(s.kv.attend(0, q, s.batch, block_length=32), first)
    lens = torch.tensor([rows, rows], dtype=torch.int32, device="cuda")
    batch = dm.KVBatch(s.batch.tensors[0], s.batch.tensors[1], lens, rows)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.kv.attend(0, q, batch, block_length=32, out=out, lse=lse)
        s.kv.attend(0, q, batch, block_length=32, out=out, lse=lse)
    for want in ([rows, rows], [rows + 33, 1200], s.lens):
        lens.copy_(torch.tensor(want, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        verify_attend(s, q, "bf16", 32, out, lse, lens=want, rows=6)
    assert torch.equal(out, first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    a = s.kv.attend(0, q, s.batch, block_length=32, stream=side.cuda_stream)
    b = s.kv.attend(0, q, s.batch, block_length=32)  # at the same time
    side.synchronize()
    torch.cuda.synchronize()
    assert torch.equal(a, first) and torch.equal(b, first)
    s.kv.check()


def gpu_values(s, which, i, n):
    """held() as a float64 tensor on the GPU [n, heads_kv, d]."""
    t = getattr(s.kv, which)[0]
    p = torch.arange(n, device="cuda")
    pg, of = torch.from_numpy(s.table[i].astype(np.int64)).cuda()[p // s.page], p % s.page
    if s.kv_name != "e4m3":
        return t[pg, :, of].double()
    sc = getattr(s.kv, which + "_scale")[0].view(torch.uint8)[pg, :, of // 32].double()
    return t.view(torch.uint8)[pg, :, of].view(torch.float8_e4m3fn).double() * torch.exp2(sc - 127)[..., None]


@pytest.mark.gpu
@pytest.mark.parametrize("kv,q_len,block,io", [("e4m3", 32, 32, "bf16"), ("e4m3", 33, 1, "f16"), ("bf16", 32, 32, "bf16"),
                                               ("e4m3", 1, 1, "bf16"), ("f16", 2, 1, "f16")])
def test_attend_whole_batches_with_cold_caches(kv, q_len, block, io):
    """Batches that fill the GPU, every row of the output, with keys and values from memory and not from L2:
    whatever the kernel's parts are handed late must still be there when it is used."""
    s = Setup([q_len] * 12, [9000 - 600 * i + (i % 3) for i in range(12)], kv, 32, 4, 128, page=64, seed=q_len)
    g = torch.Generator(device="cuda").manual_seed(1)
    for held, scale in ((s.kv.k, s.kv.k_scale), (s.kv.v, s.kv.v_scale)):
        x = torch.randn(held.shape, generator=g, device="cuda")
        held.copy_(x.to(held.dtype))
        if kv == "e4m3":  # scales that differ from block to block
            scale.view(torch.uint8).copy_(torch.randint(121, 128, scale.shape, generator=g, device="cuda").to(torch.uint8))
    q = queries(s, io, size=0.7)
    flush = torch.empty(1 << 28, dtype=torch.uint8, device="cuda")
    outs = []
    for _ in range(4):
        flush.zero_()
        outs.append(s.kv.attend(0, q, s.batch, block_length=block))
    s.kv.check()
    assert all(torch.equal(o, outs[0]) for o in outs[1:])
    verify_on_gpu(s, q, io, block, outs[0])


def verify_on_gpu(s, q, io, block, out):
    """Every row of the output against torch in float64."""
    kv, group = s.kv_name, s.nh // s.nk
    for i, (a, n) in enumerate(zip(s.q_lens, s.lens)):
        if a == 0:
            continue
        k, v = gpu_values(s, "k", i, n), gpu_values(s, "v", i, n)
        x = q[s.start[i]:s.start[i] + a].double().view(a, s.nk, group, s.d)
        pos = torch.arange(n - a, n, device="cuda")
        sees = torch.arange(n, device="cuda")[None, :] // block <= (pos // block)[:, None]
        score = torch.einsum("ahgd,nhd->ahgn", x, k) * s.d ** -0.5
        w = torch.softmax(score.masked_fill(~sees[:, None, None, :], -float("inf")), -1)
        ref = torch.einsum("ahgn,nhd->ahgd", w, v)
        size = torch.einsum("ahgn,nhd->ahgd", w, v.abs())
        err = (out[s.start[i]:s.start[i] + a].double().view_as(ref) - ref).abs()
        # as attend_tolerance: the weights' half step, the scores' errors (sums of d + 16 additions that may truncate, a
        # query rounded to bf16 on bf16 pages) twice, the sums over the positions, the output's half step. The smallest
        # step of f16 weights: 2^-25 of the largest weight times value scale, over n positions of at most 448 (e4m3)
        bf = kv == "bf16"
        dot = float(torch.einsum("ahgd,nhd->ahgn", x.abs(), k.abs()).max()) * s.d ** -0.5
        ds = dot * ((s.d + 16) * 2.0 ** -23 + 2.0 ** -21 + (kv_ref.HALF_STEP["bf16"] if bf and io == "f16" else 0.0))
        rel = kv_ref.HALF_STEP["bf16" if bf else "f16"] + 2 * np.expm1(ds + 2.0 ** -21) + (n / 8 + 64) * 2.0 ** -23
        spread = 2.0 ** 6 if kv == "e4m3" else 1.0  # of the value scales
        floor = 0.0 if bf else 2.0 ** -25 * float(w.max()) * n * float(v.abs().max()) * spread
        tol = rel * size + kv_ref.HALF_STEP[io] * ref.abs() * 1.01 + floor + 2.0 ** -25
        assert bool((err <= tol).all()), (i, float((err / tol).max()))


@pytest.mark.gpu
@pytest.mark.parametrize("kv,heads_kv,dim", [("e4m3", 2, 128), ("bf16", 2, 64), ("f16", 4, 128)])
def test_attend_many_unequal_sequences(kv, heads_kv, dim):
    """Several items to a CTA, one after the other, of one and of two 128-row halves in any order."""
    rng = np.random.default_rng(dim)
    q_lens = rng.integers(1, 75, 170)
    s = Setup(q_lens, rng.integers(0, 300, 170), kv, 16, heads_kv, dim, page=32, seed=7)
    g = torch.Generator(device="cuda").manual_seed(2)
    for held, scale in ((s.kv.k, s.kv.k_scale), (s.kv.v, s.kv.v_scale)):
        held.copy_(torch.randn(held.shape, generator=g, device="cuda").to(held.dtype))
        if kv == "e4m3":
            scale.view(torch.uint8).copy_(torch.randint(121, 128, scale.shape, generator=g, device="cuda").to(torch.uint8))
    q = queries(s, "bf16", size=0.7)
    out = s.kv.attend(0, q, s.batch, block_length=1)
    for _ in range(5):
        assert torch.equal(s.kv.attend(0, q, s.batch, block_length=1), out)
    s.kv.check()
    verify_on_gpu(s, q, "bf16", 1, out)


# ------------------------------------------------------------------------------------------------
# append
# ------------------------------------------------------------------------------------------------
def append_and_check(s, io, q_io=None, rot=64, base=10000.0, norm=True, qkv=None, q_out=None, batch=None, lens=None):
    """One append against the restatement: queries, codes (or values) and scales of every position."""
    lens = s.lens if lens is None else lens
    g = torch.Generator(device="cuda").manual_seed(int(s.rng.integers(1 << 30)))
    width = (s.nh + 2 * s.nk) * s.d
    if qkv is None:
        qkv = (torch.randn(s.rows, width, generator=g, device="cuda") *
               torch.exp(0.5 * torch.randn(width, generator=g, device="cuda"))).to(TORCH[io])
    w = [1 + 0.2 * torch.randn(s.d, generator=g, device="cuda") for _ in "qk"] if norm else [None, None]
    before = {n: [getattr(s, "held")(n, i, m) for i, m in enumerate(lens)] for n in "kv"}
    raw = {n: getattr(s.kv, n).view(torch.uint8).clone() for n in "kv"}
    if q_out is None:
        q_out = torch.full((s.rows, s.nh, s.d), 7.0, device="cuda", dtype=TORCH[q_io or io])
    got = s.kv.append(0, qkv, batch or s.batch, n_head=s.nh, q_norm=w[0], k_norm=w[1], eps=EPS, rotary_dim=rot,
                      rope_base=base, q_out=q_out)
    assert got is q_out
    s.kv.check()
    assert bool((q_out[s.n:] == 7.0).all())
    wn = [None if x is None else x.double().cpu().numpy() for x in w]
    written = {n: np.zeros((s.n_pages, s.page), bool) for n in "kv"}
    for i, (a, n) in enumerate(zip(s.q_lens, lens)):
        if a == 0:
            continue
        x = qkv[s.start[i]:s.start[i] + a].double().cpu().numpy().reshape(a, s.nh + 2 * s.nk, s.d)
        pad = max(0, a - n)
        qg = q_out[s.start[i]:s.start[i] + a].double().cpu().numpy()
        assert (qg[:pad] == 0).all()
        x, qg = x[pad:], qg[pad:]
        if len(x) == 0:
            continue
        pos = np.arange(max(0, n - a), n)
        ref = kv_ref.norm_rotate(x[:, :s.nh], wn[0], pos, rot, base, EPS)
        qi = q_io or io
        tol = kv_ref.HALF_STEP[qi] * np.abs(ref) * 1.001 + kv_ref.ROTATE_ERR * kv_ref.pair_norm(ref, rot) + (2.0 ** -25 if qi == "f16" else 0)
        err = np.abs(qg - ref)
        assert (err <= tol).all(), float((err / np.maximum(tol, 1e-300)).max())
        new_k = kv_ref.norm_rotate(x[:, s.nh:s.nh + s.nk], wn[1], pos, rot, base, EPS)
        new_v = x[:, s.nh + s.nk:]
        for name, new, slack in (("k", new_k, kv_ref.ROTATE_ERR * kv_ref.pair_norm(new_k, rot)), ("v", new_v, 0.0 * new_v)):
            now, unit = s.held(name, i, n)
            at = pos[0]
            if s.kv_name != "e4m3":
                err = np.abs(now[at:] - new)
                tol = kv_ref.HALF_STEP[s.kv_name] * np.abs(new) * 1.001 + slack + (2.0 ** -25 if s.kv_name == "f16" else 0)
                assert (err <= tol).all(), (name, float((err / np.maximum(tol, 1e-300)).max()))
                assert np.array_equal(now[:at], before[name][i][0][:at])
            else:
                assert np.array_equal(now[:at // 32 * 32], before[name][i][0][:at // 32 * 32])
                full = np.concatenate([before[name][i][0][:at], new])
                slk = np.concatenate([np.zeros((at, s.nk, s.d)), slack])
                for b in range(at // 32 * 32, n, 32):
                    for h in range(s.nk):
                        x_b, s_b = full[b:b + 32, h], slk[b:b + 32, h]
                        e = kv_ref.exponent(np.abs(x_b).max())
                        gu = unit[b, h]
                        border = [kv_ref.exponent(np.abs(x_b).max() * f) for f in (1 - 2.0 ** -18, 1 + 2.0 ** -18)]
                        assert gu in (2.0 ** e, *(2.0 ** y for y in border)), (name, i, b, h, gu, e)
                        y = now[b:b + 32, h]
                        near = kv_ref.HALF_STEP["e4m3"] * (np.abs(x_b) + s_b) + 2.0 ** -10 * gu + s_b
                        assert (np.abs(y - x_b) <= near).all(), (name, i, b, h)
                        if name == "v" or not np.any(s_b):  # nothing was computed: exactly the nearest code
                            assert np.array_equal(y, kv_ref.DECODE[kv_ref.encode(x_b / gu)] * gu)
            written[name][s.table[i, np.arange(at // 32 * 32, n) // s.page], np.arange(at // 32 * 32, n) % s.page] = True
    for name in "kv":  # nothing else changed
        now = getattr(s.kv, name).view(torch.uint8)
        same = (now == raw[name]).flatten(4).all(-1)[0].all(1).cpu().numpy()  # [page, position]
        assert same[~written[name]].all()
    return qkv, q_out


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["e4m3", "bf16", "f16"])
@pytest.mark.parametrize("io,q_io", [("f32", "bf16"), ("bf16", "bf16"), ("f16", "f32"), ("f32", "f32")])
@pytest.mark.parametrize("heads,heads_kv,dim,rot", [(8, 2, 128, 64), (4, 2, 64, 32), (3, 3, 128, 128), (6, 1, 64, 0), (4, 1, 64, 16)])
def test_append(kv, io, q_io, heads, heads_kv, dim, rot):
    s = Setup([1, 32, 33, 5, 70, 1], [0, 64, 31, 30, 95, 1000], kv, heads, heads_kv, dim, page=96, seed=rot, spare_rows=2)
    append_and_check(s, io, q_io, rot=rot, norm=rot != 32)


@pytest.mark.gpu
def test_append_many_single_tokens():
    s = Setup([1] * 75, [(37 * i) % 211 for i in range(75)], "e4m3", 8, 2, 128, page=32, seed=1)
    append_and_check(s, "bf16")


@pytest.mark.gpu
def test_append_long_prompt_and_far_positions():
    s = Setup([1111, 3], [0, 3], "e4m3", 8, 2, 128, page=128, seed=1)
    append_and_check(s, "bf16", base=600000.0)
    s = Setup([2], [299999], "e4m3", 2, 1, 64, page=4096, seed=1, fill=False)
    s.kv.k.view(torch.uint8).zero_(), s.kv.v.view(torch.uint8).zero_()
    s.kv.k_scale.view(torch.uint8).fill_(67), s.kv.v_scale.view(torch.uint8).fill_(67)
    append_and_check(s, "f32", rot=64, base=600000.0)


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["e4m3", "bf16"])
def test_append_padding_and_empty(kv):
    s = Setup([4, 0, 40, 3], [0, 0, 0, 0], kv, 8, 2, 64, page=32, seed=9, spare_rows=4)
    lens = [0, 0, 33, 1]
    append_and_check(s, "bf16", rot=32, batch=s.make_batch(lens), lens=lens)


@pytest.mark.gpu
def test_append_strides():
    s = Setup([3, 37], [100, 7], "e4m3", 8, 2, 128, seed=2, spare_rows=1)
    width = 12 * 128
    for at in (8, 3):
        wide = torch.randn(s.rows, width + 40, device="cuda")
        buf = torch.full((s.rows, 8 * 128 + 16), 7.0, device="cuda", dtype=torch.bfloat16)
        append_and_check(s, "f32", "bf16", qkv=wide[:, at:at + width], q_out=buf[:, at:at + 1024].unflatten(1, (8, 128)))
        assert bool((buf[:, :at] == 7.0).all()) and bool((buf[:, at + 1024:] == 7.0).all())


@pytest.mark.gpu
def test_append_scale_grows_and_shrinks():
    """Values that a block keeps move to a larger scale as a large row arrives, and back when it is replaced."""
    s = Setup([1], [40], "e4m3", 4, 2, 64, page=64, seed=3)
    width = 8 * 64
    big = torch.randn(1, width, device="cuda") * 100.0
    before = s.kv.v_scale.view(torch.uint8).clone()
    append_and_check(s, "f32", rot=0, norm=False, qkv=big)
    assert bool((s.kv.v_scale.view(torch.uint8)[0, int(s.table[0, 0]), :, 1] > before[0, int(s.table[0, 0]), :, 1]).all())
    append_and_check(s, "f32", rot=0, norm=False, qkv=big * 1e-4)
    append_and_check(s, "f32", rot=0, norm=False, qkv=big * 0.0)
    append_and_check(s, "f32", rot=0, norm=False, qkv=big * 1e30)
    append_and_check(s, "f32", rot=0, norm=False, qkv=big * 1e-30)


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["e4m3", "bf16"])
def test_append_not_finite(kv):
    s = Setup([33], [32], kv, 4, 2, 64, page=32, seed=3)
    qkv = torch.randn(33, 8 * 64, device="cuda")
    for r, c, x in ((3, 4 * 64 + 2, float("inf")), (32, 6 * 64 + 9, float("-inf")), (5, 7 * 64 + 1, float("nan"))):
        qkv[r, c] = x
    s.kv.append(0, qkv, s.batch, n_head=4)
    k, _ = s.held("k", 0, 65)
    v, vu = s.held("v", 0, 65)
    want_k, want_v = np.zeros(k.shape, bool), np.zeros(v.shape, bool)
    want_k[32 + 3, 0, 2] = want_v[32 + 32, 0, 9] = want_v[32 + 5, 1, 1] = True
    assert np.array_equal(~np.isfinite(k), want_k) and np.array_equal(~np.isfinite(v), want_v)
    if kv == "e4m3":
        assert np.isnan(k[35, 0, 2]) and np.isnan(v[64, 0, 9])
    fin = ~want_v[32:]
    x = qkv[:, 6 * 64:].double().cpu().numpy().reshape(33, 2, 64)[fin]
    # e4m3's smallest half step is 2^-10 of the block's scale 2^e: 2^-17 at e = -7 (amax up to 448 * 2^-7 = 3.5), but
    # normal values reach past 3.5 in 4222 draws, where e = -6 and the half step is 2^-16
    unit = np.broadcast_to(vu[32:, :, None], v[32:].shape)[fin]
    assert (np.abs(v[32:][fin] - x) <= kv_ref.HALF_STEP[kv] * np.abs(x) + 2.0 ** -10 * unit * (kv == "e4m3")).all()


@pytest.mark.gpu
def test_bad_pages_and_batches_are_reported():
    s = Setup([3, 40, 2], [64, 30, 100], "e4m3", 8, 2, 128, page=64, seed=2)
    s.ctx = s.lens
    s.fill()
    q = queries(s, "bf16")
    good = s.kv.attend(0, q, s.batch, block_length=1).clone()
    qkv = torch.randn(s.rows, 12 * 128, device="cuda").to(torch.bfloat16)
    names = ("k", "v", "k_scale", "v_scale")
    held = {n: getattr(s.kv, n).view(torch.uint8).clone() for n in names}
    for bad in (-1, s.n_pages, 2 ** 31 - 1):
        table = s.table.copy()
        table[1, 1] = bad
        keep, s.table = s.table, table
        batch = s.make_batch(s.lens)
        s.table = keep
        out = s.kv.attend(0, q, batch, block_length=1)
        with pytest.raises(dm.DmoeError, match="page number"):
            s.kv.check()
        assert torch.equal(out[:3], good[:3]) and torch.equal(out[43:], good[43:])
        s.kv.append(0, qkv, batch, n_head=8)
        with pytest.raises(dm.DmoeError, match="page number"):
            s.kv.check()
        for n in names:
            getattr(s.kv, n).view(torch.uint8).copy_(held[n])
    for lens, start, max_q in (([64 + 3, -5, 102], s.start, 40), ([67, 1 << 20, 102], s.start, 40), (s.lens, [0, 3, 2, 45], 40),
                               (s.lens, [0, 3, 99, 45], 40), (s.lens, [-1, 3, 43, 45], 40), (s.lens, s.start, 3)):
        keep, s.start = s.start, np.asarray(start, np.int32)
        batch = s.make_batch(lens, max_q)
        s.start = keep
        s.kv.attend(0, q, batch, block_length=1)
        with pytest.raises(dm.DmoeError, match="invalid q_start"):
            s.kv.check()
        s.kv.append(0, qkv, batch, n_head=8)
        with pytest.raises(dm.DmoeError, match="invalid q_start"):
            s.kv.check()
    s.kv.check()


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["e4m3", "bf16"])
@pytest.mark.parametrize("q", [1, 32])
def test_append_then_attend(kv, q):
    """The two together, as a model uses them: positions arrive in steps and each step attends to all before."""
    s = Setup([q, q], [0, 0], kv, 8, 2, 128, page=64, seed=12)
    s.table = np.arange(2 * 4, dtype=np.int32).reshape(2, 4)
    s.kv = dm.PagedKV(n_pages=8, n_head_kv=2, head_dim=128, page_size=64, kv_type=kv)
    s.n_pages = 8
    at = [0, 0]
    for step in range(5):
        lens = [at[0] + q, at[1] + q]
        s.lens = lens
        batch = s.make_batch(lens)
        _, rot = append_and_check(s, "f32", "bf16", batch=batch, lens=lens)
        check_attend(s, rot, "bf16", 32 if q == 32 else 1, batch=batch, lens=lens, rows=8)
        at = [at[0] + q, at[1] + (q if step % 2 else 0)]  # sequence 1 writes some blocks twice


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["e4m3", "bf16"])
def test_offsets_past_32_bits(kv):
    """Pages whose bytes, elements and rows lie past 2^32: the same results as on the first pages."""
    n_pages = 40000 if kv == "e4m3" else 34000  # 8 heads x 128 positions x 128: 5.2 GB of bytes, 4.4 G elements
    cache = dm.PagedKV(n_pages=n_pages, n_head_kv=8, head_dim=128, page_size=128, kv_type=kv)
    g = torch.Generator(device="cuda").manual_seed(3)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    for rows, n_head in ((1, 8), (200, 16)):
        qkv = torch.randn(rows, (n_head + 16) * 128, generator=g, device="cuda")
        got = []
        for pages in ([0, 1], [n_pages - 1, n_pages - 2]):
            batch = cache.batch(i32([pages]), i32([0, rows]), i32([rows + 7]), rows)
            for p in pages:  # the seven positions before
                cache.k[0, p].view(torch.uint8).zero_(), cache.v[0, p].view(torch.uint8).zero_()
                if kv == "e4m3":
                    cache.k_scale.view(torch.uint8)[0, p] = 127
                    cache.v_scale.view(torch.uint8)[0, p] = 127
            q = cache.append(0, qkv, batch, n_head=n_head, rotary_dim=64, q_type=torch.bfloat16)
            got.append((q, cache.k[0, pages].view(torch.uint8).clone(), cache.v[0, pages].view(torch.uint8).clone(),
                        cache.attend(0, q, batch)))
        cache.check()
        assert all(torch.equal(a, b) for a, b in zip(*got))
        assert bool(got[0][1].any()) and bool((got[0][3] != 0).any())


@pytest.mark.gpu
def test_thousands_of_sequences():
    """More sequences than a CTA has threads, most of them of one row."""
    rng = np.random.default_rng(5)
    q_lens = np.where(rng.random(3000) < 0.02, 20, 1) * (rng.random(3000) < 0.9)
    s = Setup(q_lens, rng.integers(0, 40, 3000), "e4m3", 4, 2, 64, page=32, seed=11, fill=False)
    g = torch.Generator(device="cuda").manual_seed(2)
    for held, scale in ((s.kv.k, s.kv.k_scale), (s.kv.v, s.kv.v_scale)):
        held.copy_(torch.randn(held.shape, generator=g, device="cuda").to(held.dtype))
        scale.view(torch.uint8).fill_(126)
    _, rot = append_and_check(s, "f32", "bf16", rot=32)
    out = s.kv.attend(0, rot, s.batch)
    s.kv.check()
    verify_on_gpu(s, rot, "bf16", 1, out)

"""Measured cases of the paged key/value cache: appending to it and attending over it.

"append": the fused projections [n, (n_head + 2 n_head_kv) head_dim] of a batch of sequences get the
RMS norm of each query and key head, the partial NeoX rotation at their positions, and their keys and
values are written into the cache's pages; the rotated queries come back. "attend": softmax attention
of those queries over the pages, key j visible to position i iff j / block <= i / block (block 1 is
causal), query head h reading key/value head h / (n_head / n_head_kv).

A cache is held in bf16, in f16, or in 8 bits: e4m3 values with one power-of-two scale for every 32
positions of a head (the smallest 2^e, -60 <= e <= 120, with amax <= 448 * 2^e).
"""
import math
import os
import sys

import torch

own = False

DEVICE = "cuda"
BLOCK = 32                      # positions that share a scale
E_MIN, E_MAX = -60, 120
EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
QUERY = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.bfloat16}  # projections' type -> queries' type


# ------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------
def listed():
    flash = dict(heads=32, heads_kv=4, dim=128, rot=64, base=600000.0)
    tiny = dict(heads=4, heads_kv=2, dim=64, rot=32, base=10000.0)
    return [
        # one denoising step of one sequence: its 32-position block is written again at every step
        dict(name="append one block", op="append", kv="e4m3", io="f32", n_seq=1, q=32, ctx_lo=4064, ctx_hi=4064,
             ragged=False, page=64, block=32, **flash),
        # 64 sequences that each gain one position inside a scale block (the kept part may be rescaled)
        dict(name="append 64 single tokens", op="append", kv="e4m3", io="bf16", n_seq=64, q=1, ctx_lo=101,
             ctx_hi=8003, ragged=False, page=64, block=1, **flash),
        # the first steps of the next block (previous block and this one) of 24 sequences, 16-bit cache
        dict(name="append 24 first steps", op="append", kv="bf16", io="bf16", n_seq=24, q=64, ctx_lo=480,
             ctx_hi=7904, ragged=False, page=32, block=32, **flash),
        # a long prompt enters the cache at once
        dict(name="append prompt 16384", op="append", kv="e4m3", io="bf16", n_seq=1, q=16384, ctx_lo=0, ctx_hi=0,
             ragged=False, page=128, block=32, **flash),
        # the smallest calls: one token of one short sequence, where latency counts
        dict(name="attend token 500", op="attend", kv="e4m3", io="bf16", n_seq=1, q=1, ctx_lo=499, ctx_hi=499,
             ragged=False, page=64, block=1, **flash),
        # one token of one sequence with a long context, 8-bit
        dict(name="attend token 131072", op="attend", kv="e4m3", io="bf16", n_seq=1, q=1, ctx_lo=131071,
             ctx_hi=131071, ragged=False, page=64, block=1, **flash),
        # a serving batch: 64 sequences of unequal length, one token each
        dict(name="attend 64 tokens ragged", op="attend", kv="e4m3", io="bf16", n_seq=64, q=1, ctx_lo=1001,
             ctx_hi=16001, ragged=False, page=64, block=1, **flash),
        # one denoising step of one sequence: 32 queries see each other and the whole past
        dict(name="attend block 4096", op="attend", kv="e4m3", io="bf16", n_seq=1, q=32, ctx_lo=4064, ctx_hi=4064,
             ragged=False, page=64, block=32, **flash),
        # a batch of denoising steps over unequal pasts
        dict(name="attend 16 blocks ragged", op="attend", kv="e4m3", io="bf16", n_seq=16, q=32, ctx_lo=512,
             ctx_hi=16352, ragged=False, page=64, block=32, **flash),
        # a whole prompt, block-causal
        dict(name="attend prompt 4096", op="attend", kv="e4m3", io="bf16", n_seq=1, q=4096, ctx_lo=0, ctx_hi=0,
             ragged=False, page=128, block=32, **flash),
        # one chunk of a long prompt over a 16-bit cache of what went before
        dict(name="attend chunk 2048 of 16384", op="attend", kv="bf16", io="bf16", n_seq=1, q=2048, ctx_lo=14336,
             ctx_hi=14336, ragged=False, page=64, block=32, **flash),
        # the small test model's heads, causal, odd lengths
        dict(name="attend 5 small ragged", op="attend", kv="f16", io="f16", n_seq=5, q=77, ctx_lo=3, ctx_hi=1211,
             ragged=True, page=32, block=1, **tiny),
    ]


def log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend"])
    shape = rng.choice([dict(heads=32, heads_kv=4, dim=128, rot=64, base=600000.0)] * 2 +
                       [dict(heads=4, heads_kv=2, dim=64, rot=32, base=10000.0),
                        dict(heads=16, heads_kv=16, dim=128, rot=128, base=10000.0),
                        dict(heads=24, heads_kv=8, dim=64, rot=64, base=500000.0)])
    case = dict(op=op, kv=rng.choice(["e4m3", "e4m3", "bf16", "f16"]), io=rng.choice(["bf16", "bf16", "f16"] + ["f32"] * (op == "append")),
                page=rng.choice([32, 64, 96, 128]), **shape)
    while True:
        kind = rng.choice(["token", "block", "prompt"])
        n_seq = log_int(rng, 1, 4) if kind == "prompt" else log_int(rng, 1, 64)
        q = {"token": rng.choice([1, 1, 1, 2, 3]), "block": rng.choice([16, 32, 33, 64]),
             "prompt": log_int(rng, 100, 8192)}[kind]
        lo = log_int(rng, 1, 16000) - 1
        hi = max(lo, log_int(rng, 1, 16000))
        c = dict(case, n_seq=n_seq, q=q, ctx_lo=lo, ctx_hi=hi, ragged=rng.random() < 0.5 and q > 1,
                 block=1 if kind == "token" else rng.choice([1, 32]))
        tokens = n_seq * (hi + q)
        pairs = n_seq * q * (hi + q) * c["heads"]
        if op == "append" and n_seq * q * (c["heads"] + 2 * c["heads_kv"]) * c["dim"] <= 80e6 and tokens <= 6e5:
            return c
        if op == "attend" and pairs <= 1.0e9 and tokens * c["heads_kv"] * c["dim"] <= 3e8:
            return c


def lengths(c):
    """(queries, positions before them) of each sequence."""
    n = c["n_seq"]
    ctx = [c["ctx_lo"] + (c["ctx_hi"] - c["ctx_lo"]) * ((i * 5) % n) // max(1, n - 1) for i in range(n)]
    q = [1 + (c["q"] - 1) * (1 + (i * 7 + 3) % n) // n if c["ragged"] else c["q"] for i in range(n)]
    return q, ctx


def work(c):
    q, ctx = lengths(c)
    n, nh, nk, d = sum(q), c["heads"], c["heads_kv"], c["dim"]
    io, held = (4 if c["io"] == "f32" else 2), (1 if c["kv"] == "e4m3" else 2)  # bytes of a projection and of a held value
    if c["op"] == "append":
        kept = sum(x % BLOCK for x in ctx) if c["kv"] == "e4m3" else 0
        blocks = sum((x + y - 1) // BLOCK - x // BLOCK + 1 for x, y in zip(ctx, q)) if c["kv"] == "e4m3" else 0
        return {"bytes": n * ((nh + 2 * nk) * io + nh * 2) * d + 2 * nk * (n + kept) * d * held + 2 * nk * blocks,
                "flops": 10 * n * (nh + 2 * nk) * d}
    seen = 0
    for a, x in zip(q, ctx):
        if c["block"] == 1:
            seen += a * x + a * (a + 1) // 2
        else:
            seen += sum(min(a + x, (x + i) // c["block"] * c["block"] + c["block"]) for i in range(a))
    total = sum(q) + sum(ctx)
    scales = 2 * nk * sum((a + x + BLOCK - 1) // BLOCK for a, x in zip(q, ctx)) if c["kv"] == "e4m3" else 0
    return {"bytes": 2 * n * nh * d * io + 2 * total * nk * d * held + scales, "flops": 4 * seen * nh * d}


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def exponent(amax):
    """The smallest e in [E_MIN, E_MAX] with amax <= 448 * 2^e (448 = 0.875 * 2^9), elementwise."""
    m, x = torch.frexp(amax)
    e = torch.where(m <= 0.875, x - 9, x - 8)
    return torch.where(amax > 0, e, torch.full_like(e, E_MIN)).clamp(E_MIN, E_MAX)


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    q, ctx = lengths(c)
    n, nh, nk, d, page, n_seq = sum(q), c["heads"], c["heads_kv"], c["dim"], c["page"], c["n_seq"]
    pages = [-(-(a + x) // page) for a, x in zip(q, ctx)]
    n_pages = sum(pages) + 3

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEVICE)

    order = torch.randperm(n_pages, generator=g, device=DEVICE).to(torch.int32)
    table = torch.full((n_seq, max(pages)), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for i, m in enumerate(pages):
        table[i, :m] = order[at:at + m]
        at += m
    starts = [sum(q[:i]) for i in range(n_seq + 1)]
    s = dict(case=c, table=table, q_start=torch.tensor(starts, dtype=torch.int32, device=DEVICE),
             kv_len=torch.tensor([a + x for a, x in zip(q, ctx)], dtype=torch.int32, device=DEVICE))
    # what the cache holds: keys with channels of unequal size, values whose size varies by token
    shape = (n_pages, nk, page, d)
    held = torch.float8_e4m3fn if c["kv"] == "e4m3" else TYPES[c["kv"]]
    if own:
        sys.path.insert(0, os.path.join(os.getcwd(), "diffuse-cpp_b200"))
        import diffuse_moe as dm

        kv = dm.PagedKV(n_pages=n_pages, n_head_kv=nk, head_dim=d, page_size=page, kv_type=c["kv"], device=DEVICE)
        s["kv"] = kv
        s["batch"] = dm.KVBatch(table, s["q_start"], s["kv_len"], max_q_len=max(q))
        s["k"], s["v"] = kv.k[0], kv.v[0]
        s["k_scale"], s["v_scale"] = (kv.k_scale[0], kv.v_scale[0]) if c["kv"] == "e4m3" else (None, None)
    else:
        s["k"], s["v"] = (torch.empty(shape, dtype=held, device=DEVICE) for _ in "kv")
        s["k_scale"], s["v_scale"] = (
            torch.empty(n_pages, nk, page // BLOCK, dtype=torch.uint8, device=DEVICE).view(torch.float8_e8m0fnu)
            if c["kv"] == "e4m3" else None for _ in "kv")
    channel = torch.exp(0.4 * normal(nk, 1, d))
    step = max(1, (1 << 26) // (nk * page * d))
    for p in range(0, n_pages, step):
        m = min(step, n_pages - p)
        for name in "kv":
            x = normal(m, nk, page, d)
            x = x * channel if name == "k" else x * torch.exp(0.5 * normal(m, nk, page, 1))
            if c["kv"] == "e4m3":
                b = x.view(m, nk, page // BLOCK, BLOCK, d)
                e = exponent(b.abs().amax((-1, -2)))
                s[name][p:p + m] = torch.ldexp(b, -e[..., None, None]).view(m, nk, page, d).to(held)
                s[name + "_scale"].view(torch.uint8)[p:p + m] = (e + 127).to(torch.uint8)
            else:
                s[name][p:p + m] = x.to(held)
    io = TYPES[c["io"]]
    if c["op"] == "append":
        s["qkv"] = (normal(n, (nh + 2 * nk) * d) * torch.exp(0.3 * normal((nh + 2 * nk) * d))).to(io)
        s["q_norm"], s["k_norm"] = (1.0 + 0.1 * normal(d) for _ in "qk")
    else:
        s["q"] = (1.5 * normal(n, nh, d)).to(io)
    return s


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------
def run(state):
    s, c = state, state["case"]
    if c["op"] == "append":
        q = (own_append if own else plain_append)(s)
        out = {"q": q, "k": s["k"], "v": s["v"]}
        return {**out, "k_scale": s["k_scale"], "v_scale": s["v_scale"]} if c["kv"] == "e4m3" else out
    return (own_attend if own else plain_attend)(s)


def own_append(s):
    c = s["case"]
    return s["kv"].append(0, s["qkv"], s["batch"], n_head=c["heads"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS,
                          rotary_dim=c["rot"], rope_base=c["base"], q_type=QUERY[c["io"]])


def own_attend(s):
    return s["kv"].attend(0, s["q"], s["batch"], block_length=s["case"]["block"])


def rows(s, n):
    """The sequence and the position of each of the n query rows."""
    seq = torch.searchsorted(s["q_start"][1:], torch.arange(n, device=s["q_start"].device, dtype=torch.int32), right=True)
    begin = s["q_start"].long()
    q_len = begin[1:] - begin[:-1]
    return seq, (s["kv_len"].long() - q_len)[seq] + torch.arange(n, device=seq.device) - begin[seq]


def rotate(x, pos, rot, base):
    half = rot // 2
    inv = base ** (-torch.arange(half, device=x.device, dtype=torch.float64) * 2.0 / rot)
    turns = pos.double()[:, None] * (inv / (2.0 * math.pi))[None, :]
    ang = (turns - turns.floor()) * (2.0 * math.pi)
    cos, sin = ang.cos().float()[:, None, :], ang.sin().float()[:, None, :]
    a, b, rest = x[..., :half], x[..., half:rot], x[..., rot:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], dim=-1)


def rms(x, w):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w


def plain_append(s):
    c = s["case"]
    nh, nk, d, page = c["heads"], c["heads_kv"], c["dim"], c["page"]
    n = s["qkv"].shape[0]
    seq, pos = rows(s, n)
    x = s["qkv"].float().view(n, nh + 2 * nk, d)
    q = rotate(rms(x[:, :nh], s["q_norm"]), pos, c["rot"], c["base"])
    k = rotate(rms(x[:, nh:nh + nk], s["k_norm"]), pos, c["rot"], c["base"])
    v = x[:, nh + nk:]
    pg = s["table"].long()[seq, pos // page]
    if c["kv"] != "e4m3":
        s["k"][pg, :, pos % page] = k.to(s["k"].dtype)
        s["v"][pg, :, pos % page] = v.to(s["v"].dtype)
        return q.to(QUERY[c["io"]])
    # every block of 32 positions that gains some: [sequence, block], one more block than the queries fill
    n_seq, width = c["n_seq"], (c["q"] + 2 * BLOCK - 2) // BLOCK
    q_len = (s["q_start"][1:] - s["q_start"][:-1]).long()
    first = (s["kv_len"].long() - q_len) // BLOCK
    p = (first[:, None] + torch.arange(width, device=pos.device))[:, :, None] * BLOCK + torch.arange(BLOCK, device=pos.device)
    live = p < s["kv_len"].long()[:, None, None]          # [sequence, block, place in the block]
    fresh = live & (p >= (s["kv_len"].long() - q_len)[:, None, None])
    pages = s["table"].long().gather(1, (p // page).flatten(1).clamp(max=s["table"].shape[1] - 1)).view_as(p).clamp(min=0)
    row = (s["q_start"][:-1].long()[:, None, None] + p - (s["kv_len"].long() - q_len)[:, None, None]).clamp(0, n - 1)
    block = pos // BLOCK - first[seq]                       # each new row's block, counted from its sequence's first
    spot = (p[..., 0] % page) // BLOCK
    for name, new in (("k", k), ("v", v)):
        codes, scale = s[name].view(torch.uint8), s[name + "_scale"].view(torch.uint8)
        raw = codes[pages, :, p % page]                                                        # [sequence, block, place, head, d]
        e_old = scale[pages[..., 0], :, spot].int() - 127                                      # [sequence, block, head]
        x = torch.where(fresh[..., None, None], new[row], torch.ldexp(raw.view(torch.float8_e4m3fn).float(), e_old[:, :, None, :, None]))
        x = torch.where(live[..., None, None], x, torch.zeros_like(x))
        e = exponent(x.abs().amax((2, 4)))
        y = torch.ldexp(x, -e[:, :, None, :, None]).to(torch.float8_e4m3fn).view(torch.uint8)
        y = torch.where(live[..., None, None], y, raw)
        codes[pages[:, 0], :, p[:, 0] % page] = y[:, 0]     # a sequence's first block holds what was kept
        codes[pg, :, pos % page] = y[seq, block, pos % BLOCK]
        scale[pg, :, (pos % page) // BLOCK] = (e + 127).to(torch.uint8)[seq, block]
    return q.to(QUERY[c["io"]])


def plain_attend(s):
    c = s["case"]
    nh, nk, d, page, n_seq = c["heads"], c["heads_kv"], c["dim"], c["page"], c["n_seq"]
    n, width = s["q"].shape[0], c["q"]
    most = s["table"].shape[1] * page
    seq, pos = rows(s, n)
    j = torch.arange(most, device=pos.device)
    pages = s["table"].long().clamp(min=0)

    def held(name):  # [sequence, head, position, d]
        x = s[name].view(torch.uint8)[pages].view(torch.float8_e4m3fn).float() if c["kv"] == "e4m3" else s[name][pages].float()
        if c["kv"] == "e4m3":
            e = s[name + "_scale"].view(torch.uint8)[pages].int() - 127
            x = torch.ldexp(x.unflatten(3, (page // BLOCK, BLOCK)), e[..., None, None]).flatten(3, 4)
        return x.transpose(1, 2).flatten(2, 3)

    place = torch.arange(n, device=pos.device) - s["q_start"].long()[seq]
    q = torch.zeros(n_seq, width, nh, d, device=pos.device)
    q[seq, place] = s["q"].float()
    q = q.view(n_seq, width, nk, nh // nk, d).permute(0, 2, 1, 3, 4).reshape(n_seq, nk, width * (nh // nk), d)
    at = torch.zeros(n_seq, width, dtype=torch.long, device=pos.device)
    at[seq, place] = pos
    limit = torch.minimum((at // c["block"] + 1) * c["block"], s["kv_len"].long()[:, None])
    limit = limit.repeat_interleave(nh // nk, 1)[:, None, :, None]
    score = (q @ held("k").transpose(2, 3)) / math.sqrt(d)
    score = score.masked_fill_(j >= limit, -math.inf)
    weight = torch.exp(score - score.amax(-1, keepdim=True))
    v = held("v").masked_fill_((j >= s["kv_len"].long()[:, None])[:, None, :, None], 0.0)
    out = (weight @ v) / weight.sum(-1, keepdim=True)
    out = out.view(n_seq, nk, width, nh // nk, d).permute(0, 2, 1, 3, 4).reshape(n_seq, width, nh, d)
    return out[seq, place].to(s["q"].dtype)


# ------------------------------------------------------------------------------------------------
# the same from the definition, in 64 bits
# ------------------------------------------------------------------------------------------------
def to_e4m3(x):
    """Nearest value of 4 exponent and 3 mantissa bits (ties to even), |x| <= 448: the step is 2^-3 of
    the value's power of two, and 2^-9 below 2^-6."""
    step = torch.ldexp(torch.ones_like(x), torch.frexp(x.abs().clamp(min=2.0 ** -6))[1] - 4)
    return torch.round(x / step) * step


def power(amax):
    """The smallest 2^e with amax <= 448 * 2^e, by counting the powers that are too small (borders are common)."""
    powers = 448.0 * torch.ldexp(torch.ones(E_MAX - E_MIN, dtype=torch.float64, device=amax.device),
                                 torch.arange(E_MIN, E_MAX, device=amax.device))
    e = E_MIN + torch.searchsorted(powers, amax.contiguous())
    return torch.ldexp(torch.ones_like(amax), e)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    nh, nk, d, page = c["heads"], c["heads_kv"], c["dim"], c["page"]
    f64 = torch.float64
    q_lens, ctxs = lengths(c)
    table = s["table"].long()
    k, v = s["k"].to(f64), s["v"].to(f64)
    if c["kv"] == "e4m3":
        ks, vs = s["k_scale"].to(f64), s["v_scale"].to(f64)

    def where(i, lo, hi):
        p = torch.arange(lo, hi, device=table.device)
        return table[i, p // page], p % page

    out, begin = [], 0
    if c["op"] == "append":
        inv = torch.tensor([c["base"] ** (-2.0 * i / c["rot"]) for i in range(c["rot"] // 2)], dtype=f64, device=table.device)
        for i, (a, x) in enumerate(zip(q_lens, ctxs)):
            t = s["qkv"][begin:begin + a].to(f64).view(a, nh + 2 * nk, d)
            begin += a
            ang = torch.arange(x, x + a, device=table.device, dtype=f64)[:, None] * inv
            turn = torch.polar(torch.ones_like(ang), ang)[:, None, :]

            def placed(y, w):
                y = y * w.to(f64) / torch.sqrt((y * y).sum(-1, keepdim=True) / d + EPS)
                h = c["rot"] // 2
                z = torch.complex(y[..., :h], y[..., h:2 * h]) * turn
                return torch.cat([z.real, z.imag, y[..., 2 * h:]], -1)

            out.append(placed(t[:, :nh], s["q_norm"]))
            new = {"k": placed(t[:, nh:nh + nk], s["k_norm"]), "v": t[:, nh + nk:]}
            if c["kv"] != "e4m3":
                pg, of = where(i, x, x + a)
                k[pg, :, of], v[pg, :, of] = new["k"], new["v"]
                continue
            lead = x % BLOCK
            pg, of = where(i, x - lead, x + a)
            nb = -(-(lead + a) // BLOCK)
            heads_of = of[::BLOCK] // BLOCK
            for held, scale, y in ((k, ks, new["k"]), (v, vs, new["v"])):
                y = torch.cat([held[pg[:lead], :, of[:lead]] * scale[pg[:lead], :, of[:lead] // BLOCK][..., None], y])
                full = torch.zeros(nb * BLOCK, nk, d, dtype=f64, device=table.device)
                full[:lead + a] = y
                unit = power(full.view(nb, BLOCK, nk, d).abs().amax((1, 3)))
                held[pg, :, of] = to_e4m3(y / unit.repeat_interleave(BLOCK, 0)[:lead + a][..., None])
                scale[pg[::BLOCK], :, heads_of] = unit
        got = {"q": torch.cat(out), "k": k, "v": v}
        return {**got, "k_scale": ks, "v_scale": vs} if c["kv"] == "e4m3" else got
    group = nh // nk
    for i, (a, x) in enumerate(zip(q_lens, ctxs)):
        q = s["q"][begin:begin + a].to(f64)
        begin += a
        pg, of = where(i, 0, a + x)
        sees = torch.arange(a + x, device=table.device)[None, :] // c["block"] <= \
            (torch.arange(x, x + a, device=table.device) // c["block"])[:, None]
        o = torch.empty(a, nh, d, dtype=f64, device=table.device)
        for h in range(nk):
            kh, vh = k[pg, h, of], v[pg, h, of]
            if c["kv"] == "e4m3":
                kh, vh = kh * ks[pg, h, of // BLOCK][:, None], vh * vs[pg, h, of // BLOCK][:, None]
            for e in range(h * group, (h + 1) * group):
                p = torch.softmax((q[:, e] @ kh.T * d ** -0.5).masked_fill(~sees, -math.inf), -1)
                o[:, e] = p @ vh
        out.append(o)
    return torch.cat(out)

"""The model over the paged cache where attention makes the logits: one block whose residual is small beside the
attention's output and whose feed-forward part is zero, so that an error of the attention is one of the logits. The limits
are below what planted mistakes (attention left out, no mask, heads exchanged, uniform weights, wrong positions) do to
the same logits, which each test asserts in the oracle. Then every forward of a generation over pages, against
the whole window."""
import math

import numpy as np
import pytest
import torch

import llada2
from test_gpu_llada2 import rel


@pytest.fixture(autouse=True)
def _need_gpu():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    torch.backends.cuda.matmul.allow_tf32 = False


def attention_model(n_layer=1):
    cfg = llada2.LLaDA2Config(n_layer=n_layer, n_embd=256, n_head=4, n_head_kv=2, head_dim=64, rotary_dim=32, n_ff=64,
                              first_k_dense=n_layer, n_vocab=1000, rope_base=10000.0, mask_token_id=999)
    w = llada2.LLaDA2Model.random_weights(cfg, seed=5)
    w["tok_embd"] *= 1e-2  # attn_norm undoes it for the attention; the residual keeps it
    for il in range(n_layer):
        b = f"blk.{il}."
        w[b + "attn_output"] *= 3.0
        w[b + "attn_q_norm"] *= 1.5  # sharper weights than uniform ones
        w[b + "ffn_down"].zero_()
    w["output"][cfg.mask_token_id] = 0.0
    return cfg, w, llada2.LLaDA2Model(cfg, w, {}, dtype=torch.float32)


def restated(cfg, w, tokens, mistake=None):
    """float64 logits of a whole window (blocks without feed-forward part)."""
    w = {k: v.double() for k, v in w.items()}
    dev, n, hd, half = tokens.device, len(tokens), cfg.head_dim, cfg.rotary_dim // 2
    pos = torch.arange(n, device=dev)
    norm = lambda x, g: x / torch.sqrt((x * x).mean(-1, keepdim=True) + cfg.rms_eps) * g  # noqa: E731

    def rope(x, at):
        ang = at[:, None, None].double() * cfg.rope_base ** (-torch.arange(half, device=dev).double() / half)
        a, b = x[..., :half], x[..., half:cfg.rotary_dim]
        return torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin(), x[..., cfg.rotary_dim:]], -1)

    x = w["tok_embd"][tokens]
    blk = pos // cfg.block_length
    for il in range(cfg.n_layer):
        b = f"blk.{il}."
        qkv = (norm(x, w[b + "attn_norm"]) @ w[b + "attn_qkv"].t()).view(n, -1, hd)
        q, k, v = qkv.split([cfg.n_head, cfg.n_head_kv, cfg.n_head_kv], 1)
        q = rope(norm(q, w[b + "attn_q_norm"]), pos + (5 if mistake == "positions" else 0))
        k = rope(norm(k, w[b + "attn_k_norm"]), pos)
        if mistake == "heads":
            v = v.flip(1)
        k, v = (t.repeat_interleave(cfg.n_head // cfg.n_head_kv, 1) for t in (k, v))
        score = torch.einsum("ihd,jhd->hij", q, k) / math.sqrt(hd) * (0.0 if mistake == "uniform" else 1.0)
        if mistake != "mask":
            score = score.masked_fill(blk[None, :] > blk[:, None], -math.inf)
        o = torch.einsum("hij,jhd->ihd", score.softmax(-1), v).reshape(n, -1) * (0.0 if mistake == "zero" else 1.0)
        x = x + o @ w[b + "attn_output"].t()
    return (norm(x, w["output_norm"]) @ w["output"].t()).cpu().numpy()


MISTAKES = ["zero", "mask", "heads", "uniform", "positions"]

# Root mean square of the attention output's relative error. A rounding with half step u is off by u / sqrt(3) of a power
# of two, and a value is 1.53 powers of two in the mean: 0.377 u. Values: 0.377 u_v. Keys: a score q.k / 8 of |q| = 12,
# |k| = 8 moves by 1.5 * 0.377 u_k, and so does its weight; queries alike. Weights and output: 0.377 u each, all
# independent. e4m3 pages (u = 2^-4, the rest bf16's 2^-8): 0.377 * sqrt(1 + 2.25) * 2^-4 = 0.0425; bf16: 0.377 * sqrt(1 +
# 2.25 + 2.25 + 2) * 2^-8 = 0.00403; f16: an eighth of that, 5.04e-4. Logits are linear in it but for the norm, which can
# only take a part out. A second block adds what the first one's error does to its queries, keys (1.5 each) and
# values: sqrt(1 + 1 + 2.25 + 2.25) = 2.55 times. The limits are three times that.
RMS = {"e4m3": 0.0425, "bf16": 4.03e-3, "f16": 5.04e-4}
LAYERS = {1: 1.0, 2: 2.55}


@pytest.mark.gpu
@pytest.mark.parametrize("kv_type", ["f16", "bf16", "e4m3"])
@pytest.mark.parametrize("n_layer", [1, 2])
def test_forward_paged_is_the_restated_attention(kv_type, n_layer):
    cfg, w, model = attention_model(n_layer)
    rng = np.random.default_rng(2)
    seqs = [torch.as_tensor(rng.integers(0, cfg.n_vocab - 1, size=n), device="cuda") for n in (96, 160)]
    kv = model.new_paged(9, kv_type, page_size=32)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    table = torch.tensor([[7, 2, 5, -1, -1], [0, 8, 1, 3, 4]], dtype=torch.int32, device="cuda")
    model.forward_paged(seqs[0][:64], kv, kv.batch(table[:1].contiguous(), i32(0, 64), i32(64), 64))
    got = model.forward_paged(torch.cat([seqs[0][64:], seqs[1]]), kv, kv.batch(table, i32(0, 32, 192), i32(96, 160), 160))
    kv.check()
    whole = lambda m=None: np.concatenate([restated(cfg, w, seqs[0], m)[64:], restated(cfg, w, seqs[1], m)])  # noqa: E731
    want, limit = whole(), 3 * RMS[kv_type] * LAYERS[n_layer]
    assert rel(got.cpu().numpy(), want) <= limit
    for m in MISTAKES:
        # sequence 0's rows are its last block, which no mask hides: sequence 1's show it
        assert rel(whole(m)[32:], want[32:]) > 1.5 * limit, m


@pytest.mark.gpu
@pytest.mark.parametrize("kv_type", ["bf16", "e4m3"])
def test_every_forward_of_a_generation(kv_type, monkeypatch):
    """Each denoising step's logits are those of the whole window as the sequence stands then."""
    cfg, w, model = attention_model(1)
    rng = np.random.default_rng(3)
    prompts = [rng.integers(0, cfg.n_vocab - 1, size=n) for n in (70, 9, 64)]
    steps, real = [], model.forward_paged

    def spy(tokens, kv, batch, **k):
        logits = real(tokens, kv, batch, **k)
        steps.append((tokens.clone(), batch.tensors[1].tolist(), batch.tensors[2].tolist(), k.get("rows"), logits))
        return logits

    monkeypatch.setattr(model, "forward_paged", spy)
    seqs, forwards = llada2.generate_batch(model, prompts, 60, steps=8, threshold=0.95, kv_type=kv_type)
    assert forwards == len(steps) and steps[0][4].shape[0] == 0
    final = {len(s): torch.as_tensor(s, device="cuda").long() for s in seqs}  # positions before a call's rows are final
    limit, n_rows = 3 * RMS[kv_type], 0
    for tokens, start, ends, rows, logits in steps[1:]:
        got = torch.full((len(tokens), cfg.n_vocab), float("nan"), device="cuda")
        got[rows if rows is not None else torch.arange(len(tokens), device="cuda")] = logits
        for i, end in enumerate(ends):
            mine = tokens[start[i]:start[i + 1]]
            # whose rows these are: the sequence that agrees with them where they are not masked
            fits = [s for s in final.values() if len(s) >= end and bool(((s[end - len(mine):end] == mine) | (mine == cfg.mask_token_id)).all())]
            assert len(fits) == 1
            window = torch.cat([fits[0][:end - len(mine)], mine])
            want = restated(cfg, w, window)[-32:]
            assert rel(got[start[i + 1] - 32:start[i + 1]].cpu().numpy(), want) <= limit, (start, ends, i)
            n_rows += 32
            if end - len(mine) > 32:
                assert rel(restated(cfg, w, window, "uniform")[-32:], want) > 1.5 * limit
    assert n_rows >= 32 * 3 * 2
    for p, s in zip(prompts, seqs):
        assert np.array_equal(s[: len(p)], p) and not np.any(s == cfg.mask_token_id)

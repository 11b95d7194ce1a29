"""The paged key/value cache's arguments, without a GPU: every refusal is a status code before any device
work; the restatement's own codec."""
import ctypes

import numpy as np
import pytest

import diffuse_moe as dm
import kv_ref

BASE = 1 << 20  # never dereferenced: the calls return before any device work


def cache(**kw):
    d = dict(k=BASE, v=BASE, k_scale=BASE, v_scale=BASE, err=BASE, n_pages=8, n_head_kv=2, head_dim=128, page_size=64,
             type=dm.TYPE_E4M3)
    d.update(kw)
    return dm.KVCacheDesc(**d)


def batch(**kw):
    d = dict(page_table=BASE, q_start=BASE, kv_len=BASE, max_pages=4, n_seq=2, max_q_len=8)
    d.update(kw)
    return dm.KVBatchDesc(**d)


def append_args(**kw):
    d = dict(qkv=BASE, q_out=BASE, q_norm=BASE, k_norm=BASE, n_tokens=16, qkv_stride=12 * 128, q_stride=8 * 128,
             qkv_type=dm.TYPE_BF16, q_type=dm.TYPE_BF16, n_head=8, rotary_dim=64, eps=1e-6, rope_base=1e4)
    d.update(kw)
    return dm.KVAppendArgs(**d)


def attention_args(**kw):
    d = dict(q=BASE, out=BASE, lse=BASE, n_tokens=16, q_stride=8 * 128, out_stride=8 * 128, type=dm.TYPE_BF16, n_head=8,
             block_length=32, scale=0.1)
    d.update(kw)
    return dm.KVAttentionArgs(**d)


def call_append(c, b, a):
    r = lambda x: None if x is None else ctypes.addressof(x)  # noqa: E731
    return dm.load().dmoe_kv_append(r(c), r(b), r(a), None)


def call_attention(c, b, a, ws=BASE, size=None):
    r = lambda x: None if x is None else ctypes.addressof(x)  # noqa: E731
    lib = dm.load()
    if size is None:
        size = lib.dmoe_kv_attention_workspace(r(c), r(b), r(a))
    return lib.dmoe_kv_attention(r(c), r(b), r(a), ws, size, None)


COMMON = [
    (dict(type=dm.TYPE_F32), {}, 2, "bf16, f16 or e4m3"),
    (dict(head_dim=96), {}, 2, "head_dim"),
    (dict(n_head_kv=3), {}, 1, "multiple of n_head_kv"),
    (dict(n_head_kv=0), {}, 1, "multiple of n_head_kv"),
    (dict(page_size=48), {}, 2, "page_size"),
    (dict(page_size=0), {}, 2, "page_size"),
    (dict(n_pages=0), {}, 1, "n_pages"),
    (dict(n_pages=1 << 31), {}, 1, "n_pages"),
    (dict(k=None), {}, 1, "null pointer"),
    (dict(v_scale=None), {}, 1, "null pointer"),
    (dict(k=BASE + 8), {}, 1, "16-byte aligned"),
    (dict(err=BASE + 2), {}, 1, "4-byte aligned"),
    ({}, dict(n_seq=-1), 1, "negative"),
    ({}, dict(max_q_len=-1), 1, "negative"),
    ({}, dict(max_pages=1 << 26), 2, "2^30"),
    ({}, dict(kv_len=None), 1, "null pointer in the batch"),
    ({}, dict(page_table=None), 1, "null pointer in the batch"),
    ({}, dict(q_start=BASE + 1), 1, "4-byte aligned"),
]


@pytest.mark.parametrize("c,b,status,text", COMMON)
def test_cache_and_batch_are_checked(c, b, status, text):
    for call, args in ((call_append, append_args()), (call_attention, attention_args())):
        assert call(cache(**c), batch(**b), args) == status
        assert text in dm.last_error(), dm.last_error()


@pytest.mark.parametrize("a,status,text", [
    (dict(qkv_type=dm.TYPE_Q8_0), 2, "f32, f16 or bf16"),
    (dict(q_type=dm.TYPE_E4M3), 2, "f32, f16 or bf16"),
    (dict(rotary_dim=8), 2, "rotary_dim"),
    (dict(rotary_dim=144), 2, "rotary_dim"),
    (dict(rotary_dim=-16), 2, "rotary_dim"),
    (dict(rope_base=0.0), 1, "rope_base"),
    (dict(rope_base=float("nan")), 1, "rope_base"),
    (dict(qkv_stride=12 * 128 - 1), 1, "shorter than a row"),
    (dict(q_stride=1), 1, "shorter than a row"),
    (dict(n_tokens=-1), 1, "negative"),
    (dict(n_tokens=1 << 31), 1, "2^31"),
    (dict(qkv=None), 1, "null pointer"),
    (dict(q_out=BASE + 1), 1, "aligned to its elements"),
    (dict(k_norm=BASE + 4), 1, "16-byte aligned"),
    (dict(n_head=7), 1, "multiple of n_head_kv"),
])
def test_append_arguments(a, status, text):
    assert call_append(cache(), batch(), append_args(**a)) == status
    assert text in dm.last_error(), dm.last_error()


@pytest.mark.parametrize("a,status,text", [
    (dict(type=dm.TYPE_F32), 2, "f16 or bf16"),
    (dict(block_length=0), 1, "block_length"),
    (dict(scale=0.0), 1, "scale"),
    (dict(scale=float("inf")), 1, "scale"),
    (dict(scale=float("nan")), 1, "scale"),
    (dict(q_stride=8 * 128 - 1), 1, "shorter than a row"),
    (dict(out_stride=0), 1, "shorter than a row"),
    (dict(out=None), 1, "null pointer"),
    (dict(q=BASE + 1), 1, "aligned to its elements"),
    (dict(lse=BASE + 2), 1, "aligned to its elements"),
    (dict(n_tokens=-1), 1, "negative"),
])
def test_attention_arguments(a, status, text):
    assert call_attention(cache(), batch(), attention_args(**a)) == status
    assert text in dm.last_error(), dm.last_error()


def test_attention_sizes_and_workspace():
    huge = dict(n_seq=1 << 20, max_q_len=1 << 20)
    assert call_attention(cache(), batch(**huge), attention_args(n_tokens=1 << 30)) == 2
    assert "n_seq * max_q_len" in dm.last_error()
    assert call_attention(cache(), batch(), attention_args(), ws=BASE + 4) == 1
    assert "16-byte aligned" in dm.last_error()
    assert call_attention(cache(), batch(), attention_args(), ws=None) == 1
    lib = dm.load()
    refs = [cache(), batch(), attention_args()]
    size = lib.dmoe_kv_attention_workspace(*(ctypes.addressof(r) for r in refs))
    assert size > 0
    assert call_attention(*refs, size=size - 1) == 1
    assert "workspace is too small" in dm.last_error()
    assert lib.dmoe_kv_attention_workspace(None, None, None) == 0


def test_nothing_to_do_and_null():
    assert call_append(cache(), batch(), append_args(n_tokens=0, qkv=None, q_out=None)) == 0
    assert call_append(cache(), batch(n_seq=0, q_start=None), append_args()) == 0
    assert call_attention(cache(), batch(), attention_args(n_tokens=0, q=None, out=None)) == 0
    assert call_attention(cache(), batch(max_q_len=0), attention_args()) == 0
    for c, b, a in ((None, batch(), 1), (cache(), None, 1), (cache(), batch(), None)):
        assert call_append(c, b, append_args() if a else None) == 1
        assert "null pointer" in dm.last_error()
        assert call_attention(c, b, attention_args() if a else None, size=1 << 30) == 1
        assert "null pointer" in dm.last_error()


def test_python_side_checks():
    import torch

    i32 = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA tensor"):
        dm.KVBatch(i32[None], i32, i32, 1)
    with pytest.raises(ValueError, match="kv_type"):
        dm.PagedKV(n_pages=1, n_head_kv=1, head_dim=64, kv_type="int4", device="cpu")
    kv = dm.PagedKV(n_pages=3, n_head_kv=2, head_dim=64, page_size=96, device="cpu")
    assert kv.k.shape == (1, 3, 2, 96, 64) and kv.k_scale.shape == (1, 3, 2, 3)
    assert kv.k.dtype == torch.float8_e4m3fn and kv.k_scale.dtype == torch.float8_e8m0fnu
    with pytest.raises(ValueError, match="rows of 512"):
        kv.append(0, torch.zeros(5, 511), None, n_head=4)
    with pytest.raises(ValueError, match="q must be"):
        kv.attend(0, torch.zeros(5, 4, 32), None)
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        kv.attend(0, torch.zeros(5, 4, 64, dtype=torch.float64), None)
    with pytest.raises(ValueError, match="q's type"):
        kv.attend(0, torch.zeros(5, 4, 64, dtype=torch.float16), None, out=torch.zeros(5, 4, 64))
    kv.check()
    kv.err.fill_(3)
    with pytest.raises(dm.DmoeError, match="page number out of range, invalid"):
        kv.check()
    kv.check()


def test_codec():
    import torch

    codes = np.arange(256, dtype=np.uint8)
    ref = torch.from_numpy(codes).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(kv_ref.DECODE, ref, equal_nan=True)
    rng = np.random.default_rng(0)
    x = np.concatenate([rng.normal(0, 1, 5000) * 2.0 ** rng.integers(-11, 7, 5000), ref[np.isfinite(ref)],
                        (kv_ref.POSITIVE[1:127] + kv_ref.POSITIVE[:126]) / 2])
    x = np.clip(x, -448, 448).astype(np.float32)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(kv_ref.encode(x.astype(np.float64)), want)
    for e in (-60, -3, 0, 9, 119):
        assert kv_ref.exponent(448.0 * 2.0 ** e) == e
        assert kv_ref.exponent(np.nextafter(448.0 * 2.0 ** e, np.inf)) == e + 1
    assert kv_ref.exponent(0.0) == -60 and kv_ref.exponent(1e300) == 120

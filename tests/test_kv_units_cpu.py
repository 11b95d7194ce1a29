"""The attention's schedule numbers its units of work in 31 bits: a call that could have more is refused."""
import diffuse_moe as dm
from test_kv_cpu import attention_args, batch, cache, call_attention


def test_units_are_counted_with_partly_filled_tiles():
    # tables of 13 pages of 32: 3.25, so 4 tiles of 128, and 4 more for each item
    c = cache(n_head_kv=8, page_size=32)
    b = dict(max_pages=13, max_q_len=17)
    a = dict(n_head=8, q_stride=8 * 128, out_stride=8 * 128, n_tokens=(1 << 31) - 1)
    for n_seq, fits in (((1 << 31) // (8 * 8) + 1, False), (35_000_000, False)):
        status = call_attention(c, batch(n_seq=n_seq, **b), attention_args(**a))
        assert (status == 0) == fits and status == 2 and "too many for one call" in dm.last_error()

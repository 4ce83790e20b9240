"""Attention over tables with room for very long rows: what the header says is served, and the refusal above it."""
import numpy as np
import pytest

from moearc_b200 import BadArgument, Context
from moearc_b200.kvcache import KvCache
from paged_model import BF16, F32, store
from test_kvcache import Described, attn, ctx, lib  # noqa: F401  (fixtures)


@pytest.mark.parametrize("kw, heads, n", [
    (dict(kv_type=0, head_dim=20, n_kv_heads=64, max_seq=1024, max_pages=1 << 20, page_tokens=1), 64, 1024),
    (dict(kv_type=30, head_dim=24, n_kv_heads=8, max_seq=1024, max_pages=1 << 24, page_tokens=127), 64, 256),
    (dict(kv_type=30, head_dim=64, n_kv_heads=8, max_seq=1024, max_pages=1 << 24, page_tokens=127), 64, 1024)])
def test_more_tiles_than_32_bits_number_are_refused(lib, ctx, kw, heads, n):  # noqa: F811
    assert n * heads * (kw["max_pages"] * kw["page_tokens"] // 8 + 2) >= 1 << 31
    stride = heads * kw["head_dim"]
    assert attn(lib, ctx, Described(**kw), heads=heads, n=n, qs=stride) == -2


@pytest.mark.gpu
@pytest.mark.parametrize("kv, D", [(F32, 20), (F32, 64), (BF16, 64)])
def test_short_rows_of_long_tables(kv, D):
    """Room for 2^28 tokens a row, just inside the limit: the same bits as with a table that fits."""
    rows, H, pt, lens = 4, 8, 64, [5, 700, 0, 64]
    assert rows * H * ((1 << 28) // 8 + 2) < 1 << 31
    rng = np.random.default_rng(D)
    with Context() as c:
        pools = [[c.upload_new(store(rng.standard_normal((20, pt, H, D), np.float32), kv))] for _ in range(2)]
        q, outs = c.upload_new(rng.standard_normal((rows, H, D), np.float32)), []
        for max_pages in (1 << 22, 11):
            cache = KvCache(c, n_layer=1, n_pages=20, page_tokens=pt, n_kv_heads=H, head_dim=D, kv_type=kv, max_seq=rows, max_pages=max_pages,
                            n_heads=H, k_pages=pools[0], v_pages=pools[1])
            cache.grow(list(range(rows)), lens)
            out = c.alloc_n(np.float32, rows * H * D)
            cache.attn_decode(0, out, q, rows, H, D ** -0.5)
            outs.append(c.download(out, np.float32, rows * H * D))
            assert cache.status() == 0
        assert np.array_equal(*outs) and np.abs(outs[0]).max() > 0
        if (kv, D) == (F32, 20):
            big = KvCache(c, n_layer=1, n_pages=20, page_tokens=pt, n_kv_heads=H, head_dim=D, kv_type=kv, max_seq=8, max_pages=1 << 23,
                          n_heads=64 * H, k_pages=pools[0], v_pages=pools[1])
            with pytest.raises(BadArgument):
                big.attn_decode(0, c.alloc_n(np.float32, 8 * 64 * H * D), c.alloc_n(np.float32, 8 * 64 * H * D), 8, 64 * H, 1.0)

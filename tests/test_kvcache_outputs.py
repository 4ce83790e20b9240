"""The buffers that a compaction may be given: both or none, and large enough, before anything is launched."""
import pytest

from moearc_b200 import BadArgument, BufferTooSmall, DeviceBuffer, kvcache


class NoDevice:
    """In a context's place: nothing below may reach the library."""
    raw = None

    def __getattr__(self, name):
        raise AssertionError(f"{name} was reached")


def cache(rows=4, max_pages=8, pages=16):
    c = object.__new__(kvcache.KvCache)
    c.ctx, c.max_seq, c.max_pages, c.n_pages = NoDevice(), rows, max_pages, pages
    c.tables, c.refs = (DeviceBuffer(c.ctx, 0x10000, n, owned=False) for n in (4 * rows * max_pages, 4 * pages))
    return c


def test_an_empty_output_is_not_the_cache_itself():
    c = cache()
    none = DeviceBuffer(c.ctx, 0x20000, 0, owned=False)
    with pytest.raises(BufferTooSmall):
        c.compact(tables_out=none, refs_out=none)
    with pytest.raises(BufferTooSmall):
        c.compact(tables_out=DeviceBuffer(c.ctx, 0x20000, 4 * 32, owned=False), refs_out=none)
    with pytest.raises(BufferTooSmall):
        c.compact(n_live=none)


def test_one_output_without_the_other_is_refused():
    c = cache()
    big = DeviceBuffer(c.ctx, 0x20000, 4096, owned=False)
    with pytest.raises(BadArgument):
        c.compact(tables_out=big)
    with pytest.raises(BadArgument):
        c.compact(refs_out=big)

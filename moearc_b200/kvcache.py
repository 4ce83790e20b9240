"""One paged KV cache for many sequences (moearc_x_kv_* and moearc_x_attn_decode_batch).

``KvCache`` names the buffers of a cache — K and V pools per layer, page tables, lengths, page
reference counts — either its own or the caller's, and has one method per call. Everything is
enqueued on the context's stream; tables, lengths and counts stay on the device, and nothing is
read back but ``status()``.

    cache = KvCache(ctx, n_layer=2, n_pages=512, page_tokens=16, n_kv_heads=8, head_dim=64,
                    kv_type=BF16, max_seq=32, max_pages=64, n_heads=64)
    cache.grow([0, 1], [5, 9])                    # rows 0 and 1 get room for 5 and 9 tokens
    cache.attn_decode(0, out, q, 2, 64, 0.125, k_new=k, v_new=v)   # stores and attends the last
    cache.fork([0], [2])                          # row 2 continues row 0
    cache.free([1])
    cache.compact()
"""
from __future__ import annotations

import ctypes as C
from array import array

import numpy as np

from . import _lib
from .kernels import KV_ELEM_BYTES, BadArgument, Context, DeviceBuffer, Failed, _p

NO_PAGE = 0xFFFFFFFF
MAX_LIST = 1024
# bits of status(): what a call without effect lacked; WAIT: a kernel's wait ran out, its output is invalid
FULL, LONG, TAKEN, WAIT = 1, 2, 4, 8


def _list(v) -> array:
    try:
        if isinstance(v, array) and v.typecode == "I":
            a = v
        elif isinstance(v, list):  # 256 rows: 3.0 us, 4.2 through the iterator
            a = array("I")
            a.fromlist(v)
        else:
            a = array("I", v)
    except (OverflowError, TypeError) as e:
        raise BadArgument(f"a row list of whole numbers is wanted: {e}") from None
    if len(a) > MAX_LIST:
        raise BadArgument(f"a list of {len(a)} rows: one call takes {MAX_LIST}")
    return a


def _at(a: array) -> int:
    return a.buffer_info()[0]


class KvCache:
    """n_heads: query heads of the attention that will read it (0: page calls only; the workspace that is
    made serves any number of them). Buffers that are not given are allocated and set up as the empty cache (``reset``); with any
    of tables, n_kv and refs given, all three are the caller's and taken as they are."""

    def __init__(self, ctx: Context, *, n_layer: int, n_pages: int, page_tokens: int, n_kv_heads: int, head_dim: int,
                 kv_type: int, max_seq: int, max_pages: int, n_heads: int = 0, k_pages: list[DeviceBuffer] | None = None,
                 v_pages: list[DeviceBuffer] | None = None, tables: DeviceBuffer | None = None,
                 n_kv: DeviceBuffer | None = None, refs: DeviceBuffer | None = None):
        if kv_type not in KV_ELEM_BYTES:
            raise BadArgument(f"KV type {kv_type}")
        if min(n_layer, n_pages, page_tokens, n_kv_heads, head_dim, max_seq, max_pages) < 1:
            raise BadArgument("a cache dimension is zero")
        given = [b is not None for b in (tables, n_kv, refs)]
        if any(given) != all(given):
            raise BadArgument("tables, n_kv and refs go together")
        self.ctx, self.n_layer, self.n_pages, self.page_tokens = ctx, n_layer, n_pages, page_tokens
        self.n_kv_heads, self.head_dim, self.kv_type, self.max_seq, self.max_pages = n_kv_heads, head_dim, kv_type, max_seq, max_pages
        self.n_heads = n_heads
        self.page_bytes = page_tokens * n_kv_heads * head_dim * KV_ELEM_BYTES[kv_type]
        pool = n_pages * self.page_bytes
        pools = []
        for what, p in (("K", k_pages), ("V", v_pages)):
            if p is not None and len(p) != n_layer:
                raise BadArgument(f"{len(p)} {what} pools for {n_layer} layers")
            for b in p or ():
                b.require(f"{what} pool", pool)
        d = _lib.KvCacheDesc(n_layer=n_layer, n_pages=n_pages, page_tokens=page_tokens, n_kv_heads=n_kv_heads, head_dim=head_dim,
                             kv_type=kv_type, max_seq=max_seq, max_pages=max_pages)
        work = ctx.lib.moearc_x_kv_work_bytes(ctx.raw, C.byref(d), n_heads)
        if not work:
            raise BadArgument("the cache's shape is not supported")
        for p in (k_pages, v_pages):
            pools.append(p if p is not None else [ctx.alloc(pool) for _ in range(n_layer)])
        self.k_pages, self.v_pages = pools
        self.tables = tables if tables is not None else ctx.alloc(4 * max_seq * max_pages)
        self.n_kv = n_kv if n_kv is not None else ctx.alloc(4 * max_seq)
        self.refs = refs if refs is not None else ctx.alloc(4 * n_pages)
        for b, what, n in ((self.tables, "page table", max_seq * max_pages), (self.n_kv, "length", max_seq), (self.refs, "reference count", n_pages)):
            b.require(what, 4 * n)
        self.work, self.flags = ctx.alloc(work), ctx.alloc(4)
        self._pools = [(C.c_void_p * n_layer)(*[b.ptr for b in p]) for p in pools]
        d.k_pages, d.v_pages = (C.cast(p, C.POINTER(C.c_void_p)) for p in self._pools)
        d.tables, d.n_kv, d.refs, d.status = self.tables.ptr, self.n_kv.ptr, self.refs.ptr, self.flags.ptr
        d.work, d.work_bytes = self.work.ptr, work
        self._desc, self._d = d, C.byref(d)
        if any(given):
            ctx.upload(self.flags, np.zeros(1, np.uint32))
        else:
            self.reset()

    def reset(self) -> None:
        """Every row empty, every page free."""
        self.ctx._finish(self.ctx.lib.moearc_x_kv_reset(self.ctx.raw, self._d), "kv_reset")

    def grow(self, seqs, add) -> None:
        """Row seqs[i] gains add[i] tokens."""
        s, a = _list(seqs), _list(add)
        if len(s) != len(a):
            raise BadArgument(f"{len(s)} rows and {len(a)} counts")
        self.ctx._finish(self.ctx.lib.moearc_x_kv_grow(self.ctx.raw, self._d, _at(s), _at(a), len(s)), "kv_grow")

    def fork(self, src, dst, deep: bool = False) -> None:
        """Empty row dst[i] becomes row src[i], sharing full pages (or, deep, copying every page; as many
        free pages as the row has table entries, holes included, have to be there)."""
        s, t = _list(src), _list(dst)
        if len(s) != len(t):
            raise BadArgument(f"{len(s)} rows to fork onto {len(t)}")
        self.ctx._finish(self.ctx.lib.moearc_x_kv_fork(self.ctx.raw, self._d, _at(s), _at(t), len(s), 1 if deep else 0), "kv_fork")

    def free(self, seqs, keep=None) -> None:
        """Row seqs[i] keeps its first keep[i] tokens (None: no tokens)."""
        s = _list(seqs)
        k = None if keep is None else _list(keep)
        if k is not None and len(s) != len(k):
            raise BadArgument(f"{len(s)} rows and {len(k)} lengths")
        self.ctx._finish(self.ctx.lib.moearc_x_kv_free(self.ctx.raw, self._d, _at(s), None if k is None else _at(k), len(s)), "kv_free")

    def compact(self, tables_out: DeviceBuffer | None = None, refs_out: DeviceBuffer | None = None,
                n_live: DeviceBuffer | None = None) -> None:
        """Moves the pages in use below every free one; tables and counts in place, or into
        tables_out and refs_out (both)."""
        if (tables_out is None) != (refs_out is None):
            raise BadArgument("tables_out and refs_out go together")
        t, r = (self.tables, self.refs) if tables_out is None else (tables_out, refs_out)
        t.require("compacted page table", 4 * self.max_seq * self.max_pages)
        r.require("compacted reference count", 4 * self.n_pages)
        if n_live is not None:
            n_live.require("live page count", 4)
        self.ctx._finish(self.ctx.lib.moearc_x_kv_compact(self.ctx.raw, self._d, t.ptr, r.ptr, _p(n_live)), "kv_compact")

    def status(self) -> int:
        """Waits; the FULL, LONG, TAKEN and WAIT bits raised since the last look (0: every call took effect)."""
        v = self.ctx.lib.moearc_x_kv_status(self.ctx.raw, self._d)
        if v < 0:
            raise Failed("kv_status failed on the device")
        return v

    def attn_decode(self, layer: int, out: DeviceBuffer, q: DeviceBuffer, n_seq: int, n_heads: int, scale: float, *,
                    q_stride: int | None = None, k_new: DeviceBuffer | None = None, v_new: DeviceBuffer | None = None,
                    new_stride: int | None = None, seqs=None, kv_begin: DeviceBuffer | None = None,
                    sinks: DeviceBuffer | None = None) -> None:
        """Attention of one new token for n_seq batch rows (moearc_x_attn_decode_batch). Strides are in
        floats; seqs names the cache rows (default 0 .. n_seq - 1)."""
        if n_heads < 1 or not self.n_heads:
            raise BadArgument(f"{n_heads} query heads (a cache made without n_heads has no workspace for attention)")
        if min(n_seq, layer, q_stride or 0, new_stride or 0) < 0:
            raise BadArgument("a negative count or stride")
        row, kv_row = n_heads * self.head_dim, self.n_kv_heads * self.head_dim
        qs = row if q_stride is None else q_stride
        ns = kv_row if new_stride is None else new_stride
        if n_seq:
            out.require("attention output", 4 * n_seq * row)
            q.require("attention query", 4 * ((n_seq - 1) * qs + row))
            for b, what in ((k_new, "new keys"), (v_new, "new values")):
                if b is not None:
                    b.require(what, 4 * ((n_seq - 1) * ns + kv_row))
            if kv_begin is not None:
                kv_begin.require("first keys", 4 * n_seq)
            if sinks is not None:
                sinks.require("sinks", 4 * n_heads)
        rows = None
        if seqs is not None:
            rows = _list(seqs)
            if len(rows) != n_seq:
                raise BadArgument(f"{len(rows)} rows for a batch of {n_seq}")
        self.ctx._finish(self.ctx.lib.moearc_x_attn_decode_batch(
            self.ctx.raw, self._d, layer, out.ptr, q.ptr, qs, _p(k_new), _p(v_new), ns, None if rows is None else _at(rows), _p(kv_begin), _p(sinks), n_seq,
            n_heads, scale), "attn_decode_batch")

"""The paged cache's host side without a GPU: refusals (before anything reaches the device), list
checks, and the host model's own rules."""
import ctypes as C

import pytest

from moearc_b200 import BadArgument, Context, _lib, kvcache
from paged_model import BF16, FULL, LONG, TAKEN, Paged

U3 = C.c_uint * 3


class Described:
    """A cache description with made-up addresses: every call below is refused before they are used."""

    def __init__(self, **kw):
        one = (C.c_void_p * 128)(*[0x10000] * 128)
        self.one = one
        v = dict(n_layer=2, n_pages=64, page_tokens=16, n_kv_heads=4, head_dim=64, kv_type=30, max_seq=8, max_pages=16,
                 tables=0x10000, n_kv=0x10000, refs=0x10000, status=0x10000, work=0x10000, work_bytes=1 << 30)
        v.update(kw)
        self.d = _lib.KvCacheDesc(**v)
        self.d.k_pages = C.cast(one, C.POINTER(C.c_void_p))
        self.d.v_pages = C.cast(one, C.POINTER(C.c_void_p))

    @property
    def ref(self):
        return C.byref(self.d)


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


@pytest.fixture(scope="module")
def ctx():
    """Zeroed bytes in the place of a context: argument checks come first and do not read it."""
    return C.create_string_buffer(4096)


BAD = [dict(n_layer=0), dict(n_layer=129), dict(n_pages=0), dict(n_pages=(1 << 28) + 1), dict(page_tokens=0), dict(n_kv_heads=0),
       dict(head_dim=0), dict(head_dim=1025), dict(kv_type=2), dict(kv_type=39), dict(max_seq=0), dict(max_seq=65537),
       dict(max_pages=0), dict(max_pages=(1 << 24) + 1), dict(max_pages=1 << 20, page_tokens=1 << 11),
       dict(page_tokens=1 << 20, max_pages=1, n_kv_heads=64, head_dim=32), dict(work=0x10008)]


@pytest.mark.parametrize("kw", BAD)
def test_a_bad_description_is_refused(lib, ctx, kw):
    k = Described(**kw)
    assert lib.moearc_x_kv_reset(ctx, k.ref) == -2
    assert lib.moearc_x_kv_grow(ctx, k.ref, U3(0, 1, 2), U3(1, 1, 1), 3) == -2
    assert lib.moearc_x_kv_fork(ctx, k.ref, U3(0, 0, 0), U3(1, 2, 3), 3, 0) == -2
    assert lib.moearc_x_kv_free(ctx, k.ref, U3(0, 1, 2), None, 3) == -2
    assert lib.moearc_x_kv_compact(ctx, k.ref, 0x10000, 0x10000, None) == -2
    assert lib.moearc_x_kv_status(ctx, k.ref) == -2
    if "work" not in kw:
        assert lib.moearc_x_kv_work_bytes(ctx, k.ref, 8) == 0


@pytest.mark.parametrize("name", ["tables", "n_kv", "refs", "status", "pool"])
def test_an_address_between_elements_is_refused(lib, ctx, name):
    for kv_type, off in ((30, 1), (0, 2)):
        k = Described(kv_type=kv_type, **({} if name == "pool" else {name: 0x10002}))
        if name == "pool":
            k.one[1] = 0x10000 + off
        assert lib.moearc_x_kv_reset(ctx, k.ref) == -2
        assert lib.moearc_x_kv_free(ctx, k.ref, U3(0, 1, 2), None, 3) == -2
        assert attn(lib, ctx, k) == -2


def test_outputs_of_a_compaction_between_elements_are_refused(lib, ctx):
    k = Described()
    for t, r, n in ((0x20002, 0x30000, None), (0x20000, 0x30001, None), (0x20000, 0x30000, 0x10002)):
        assert lib.moearc_x_kv_compact(ctx, k.ref, t, r, n) == -2


@pytest.mark.parametrize("name", ["tables", "n_kv", "refs", "status", "work"])
def test_a_missing_buffer_is_refused(lib, ctx, name):
    k = Described(**{name: None})
    assert lib.moearc_x_kv_reset(ctx, k.ref) == -1
    assert lib.moearc_x_kv_free(ctx, k.ref, U3(0, 1, 2), None, 3) == -1


def test_a_missing_pool_or_context_is_refused(lib, ctx):
    k = Described()
    k.one[1] = None
    assert lib.moearc_x_kv_reset(ctx, k.ref) == -1
    k = Described()
    assert lib.moearc_x_kv_reset(None, k.ref) == -1
    assert lib.moearc_x_kv_reset(ctx, None) == -1
    assert lib.moearc_x_kv_work_bytes(None, k.ref, 8) == 0
    assert lib.moearc_x_kv_compact(ctx, k.ref, None, 0x10000, None) == -1
    assert lib.moearc_x_kv_compact(ctx, k.ref, 0x20000, 0x10000, None) == -2  # tables elsewhere, counts in place
    assert lib.moearc_x_kv_compact(ctx, k.ref, 0x10000, 0x20000, None) == -2


def test_row_lists_are_checked(lib, ctx):
    k = Described()
    many = (C.c_uint * 1025)(*range(1025))
    assert lib.moearc_x_kv_grow(ctx, k.ref, U3(0, 1, 0), U3(1, 1, 1), 3) == -2  # the same row twice
    assert lib.moearc_x_kv_grow(ctx, k.ref, U3(0, 1, 8), U3(1, 1, 1), 3) == -2  # no such row
    assert lib.moearc_x_kv_grow(ctx, k.ref, None, U3(1, 1, 1), 3) == -1
    assert lib.moearc_x_kv_grow(ctx, k.ref, U3(0, 1, 2), None, 3) == -1
    assert lib.moearc_x_kv_grow(ctx, k.ref, many, many, 1025) == -2
    assert lib.moearc_x_kv_free(ctx, k.ref, U3(3, 3, 1), None, 3) == -2
    assert lib.moearc_x_kv_free(ctx, k.ref, many, None, 1025) == -2
    assert lib.moearc_x_kv_fork(ctx, k.ref, U3(0, 0, 0), U3(1, 2, 1), 3, 0) == -2  # onto the same row twice
    assert lib.moearc_x_kv_fork(ctx, k.ref, U3(0, 1, 0), U3(1, 2, 3), 3, 0) == -2  # from a row being made
    assert lib.moearc_x_kv_fork(ctx, k.ref, U3(0, 8, 0), U3(1, 2, 3), 3, 0) == -2
    assert lib.moearc_x_kv_fork(ctx, k.ref, U3(0, 0, 0), U3(1, 2, 8), 3, 0) == -2
    assert lib.moearc_x_kv_grow(ctx, Described(work_bytes=64).ref, U3(0, 1, 2), U3(1, 1, 1), 3) == -2
    for call in (lib.moearc_x_kv_grow, lib.moearc_x_kv_free):  # an empty list is nothing to do
        assert call(ctx, k.ref, None, None, 0) == 0
    assert lib.moearc_x_kv_fork(ctx, k.ref, None, None, 0, 1) == 0


def attn(lib, ctx, k, **kw):
    v = dict(layer=0, out=0x10000, q=0x10000, qs=512, kn=None, vn=None, ns=256, seqs=None, begin=None, sinks=None, n=4, heads=8, scale=0.125)
    v.update(kw)
    return lib.moearc_x_attn_decode_batch(ctx, k.ref, *v.values())


@pytest.mark.parametrize("kw, rc", [
    (dict(out=None), -1), (dict(q=None), -1), (dict(kn=0x10000), -1), (dict(vn=0x10000), -1), (dict(layer=2), -2), (dict(heads=0), -2),
    (dict(heads=6), -2), (dict(qs=511), -2), (dict(kn=0x10000, vn=0x10000, ns=255), -2), (dict(n=9), -2), (dict(n=1025), -2),
    (dict(seqs=U3(0, 1, 1), n=3), -2), (dict(seqs=U3(0, 1, 8), n=3), -2), (dict(scale=float("nan")), -2), (dict(scale=float("inf")), -2),
    (dict(n=0), 0)] + [({name: 0x10002, **({"kn": 0x10000, "vn": 0x10000, name: 0x10002} if name in ("kn", "vn") else {})}, -2)
                       for name in ("out", "q", "kn", "vn", "begin", "sinks")])
def test_attention_arguments_are_checked(lib, ctx, kw, rc):
    assert attn(lib, ctx, Described(), **kw) == rc


def test_more_tokens_than_the_tensor_core_kernel_numbers_are_refused(lib, ctx):
    assert attn(lib, ctx, Described(n_pages=1 << 28, page_tokens=8)) == -2
    assert attn(lib, ctx, Described(n_pages=1 << 28, page_tokens=8, kv_type=0), n=0) == 0


@pytest.mark.parametrize("kw, rc", [
    (dict(logits=None), -1), (dict(tokens=None), -1), (dict(lp=None), -1), (dict(k=2, ids=None), -1), (dict(k=2, top=None), -1),
    (dict(ty=39), -2), (dict(stride=99), -2), (dict(vocab=0), -2), (dict(k=33), -2), (dict(k=5, vocab=4), -2), (dict(scale=0.0), -2),
    (dict(scale=-1.0), -2), (dict(scale=1e-31), -2), (dict(scale=2e30), -2), (dict(scale=float("nan")), -2), (dict(scale=float("inf")), -2), (dict(logits=0x10002), -2), (dict(rows=0), 0)] +
    [({name: 0x10002, "k": 2}, -2) for name in ("tokens", "lp", "ent", "ids", "top")] + [(dict(logits=0x10001, ty=30), -2)])
def test_logprob_arguments_are_checked(lib, ctx, kw, rc):
    v = dict(logits=0x10000, ty=0, stride=100, rows=4, vocab=100, scale=1.0, tokens=0x10000, lp=0x10000, ent=0x10000, k=0, ids=0x10000, top=0x10000)
    v.update(kw)
    assert lib.moearc_x_token_logprobs(ctx, *v.values()) == rc


def test_negative_counts_and_strides_are_refused():
    """Before they would wrap to unsigned ones."""
    c = object.__new__(kvcache.KvCache)
    c.n_heads, c.head_dim, c.n_kv_heads = 8, 64, 4
    for kw in (dict(n_seq=-1), dict(layer=-1), dict(q_stride=-512), dict(new_stride=-256)):
        a = dict(layer=0, n_seq=2, q_stride=None, new_stride=None)
        a.update(kw)
        with pytest.raises(BadArgument):
            c.attn_decode(a["layer"], None, None, a["n_seq"], 8, 1.0, q_stride=a["q_stride"], new_stride=a["new_stride"])
    for kw in (dict(n_rows=-1), dict(n_vocab=-1), dict(row_stride=-100), dict(k=-1)):
        a = dict(n_rows=2, n_vocab=100, row_stride=None, k=0)
        a.update(kw)
        with pytest.raises(BadArgument):
            Context.token_logprobs(None, None, 0, a["n_rows"], a["n_vocab"], row_stride=a["row_stride"], k=a["k"])


def test_python_lists_are_checked():
    with pytest.raises(BadArgument):
        kvcache._list([0, -1])
    with pytest.raises(BadArgument):
        kvcache._list([1 << 32])
    with pytest.raises(BadArgument):
        kvcache._list(range(1025))
    with pytest.raises(BadArgument):
        kvcache._list([0.5])
    assert len(kvcache._list([])) == 0


def test_the_model_keeps_its_rules():
    m = Paged(1, 12, 4, 1, 8, BF16, 6, 5)
    m.grow([0, 1], [6, 3])
    m.check()
    m.fork([0, 0], [2, 3])
    m.check()
    assert m.tables[2][0] == m.tables[0][0] and m.tables[2][1] != m.tables[0][1] and m.row_bits(2) == m.row_bits(0)
    m.free([0, 2], [2, 2])
    m.check()
    m.grow([0], [1])  # its first page is shared: copied before it is written on
    m.check()
    assert m.tables[0][0] != m.tables[2][0] == m.tables[3][0]
    was = [m.row_bits(s)[:2] for s in range(6)]
    assert m.compact() == sum(r > 0 for r in m.refs)
    m.check()
    assert [m.row_bits(s)[:2] for s in range(6)] == was
    m.grow([1], [30])
    assert m.status == LONG
    m.fork([1], [3])
    assert m.status == LONG | TAKEN
    m.grow([1], [17])
    m.grow([4, 5], [20, 20])
    assert m.status == LONG | TAKEN | FULL
    m.check()

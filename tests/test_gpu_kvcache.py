"""The paged cache of many sequences on the B200, against the host model: page calls exactly, decode
attention of ragged batches within derived bounds, and both with token log probabilities as a
serving loop uses them."""
import numpy as np
import pytest

from moearc_b200 import BadArgument, BufferTooSmall, Context, DeviceBuffer
from moearc_b200.kvcache import FULL, LONG, NO_PAGE, TAKEN, KvCache
from paged_model import BF16, EPS, F16, F32, Paged, attend, attend_tolerance, store

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = Context()
    yield c
    c.close()


class Pair:
    """A model and a device cache in the same state; every call goes to both."""

    def __init__(self, ctx, layers=2, pages=40, pt=8, kvh=2, D=64, kv=BF16, rows=8, max_pages=12, n_heads=0, seed=0, skew=0):
        self.m = Paged(layers, pages, pt, kvh, D, kv, rows, max_pages, seed)
        self.ctx, self.layers = ctx, layers
        pools = []
        for p in (self.m.k, self.m.v):
            made = []
            for l in range(layers):
                b = ctx.alloc(p[l].nbytes + skew)
                ctx.upload(b.view(skew, p[l].nbytes), p[l])
                made.append(b.view(skew, p[l].nbytes))
                made[-1].keep = b
            pools.append(made)
        self.c = KvCache(ctx, n_layer=layers, n_pages=pages, page_tokens=pt, n_kv_heads=kvh, head_dim=D, kv_type=kv, max_seq=rows,
                         max_pages=max_pages, n_heads=n_heads, k_pages=pools[0], v_pages=pools[1])

    def do(self, name, *a, **kw):
        getattr(self.m, name)(*a, **kw)
        getattr(self.c, name)(*a, **kw)

    def put(self):
        """The model's bookkeeping onto the device."""
        for b, v in ((self.c.tables, self.m.tables), (self.c.n_kv, self.m.n_kv), (self.c.refs, self.m.refs)):
            self.ctx.upload(b, np.array(v, np.uint32))

    def same(self, pools=True):
        m, c, ctx = self.m, self.c, self.ctx
        assert ctx.download(c.n_kv, np.uint32, m.rows).tolist() == m.n_kv
        assert ctx.download(c.tables, np.uint32, m.rows * m.max_pages).reshape(m.rows, -1).tolist() == m.tables
        assert ctx.download(c.refs, np.uint32, m.pages).tolist() == m.refs
        for l in range(self.layers if pools else 0):
            for dev, host in ((c.k_pages, m.k), (c.v_pages, m.v)):
                assert np.array_equal(ctx.download(dev[l], host.dtype, host[l].size), host[l].ravel())
        assert c.status() == m.status
        m.status = 0
        m.check()


# ---- pages -------------------------------------------------------------------------------------

def test_a_new_cache_is_empty(ctx):
    p = Pair(ctx)
    p.same()
    c = KvCache(ctx, n_layer=1, n_pages=3, page_tokens=4, n_kv_heads=1, head_dim=8, kv_type=F32, max_seq=2, max_pages=2)
    assert ctx.download(c.tables, np.uint32, 4).tolist() == [NO_PAGE] * 4 and c.status() == 0


@pytest.mark.parametrize("kv, pt, D, skew", [(BF16, 8, 64, 0), (F16, 1, 3, 0), (F32, 5, 7, 0), (BF16, 3, 5, 2), (F32, 16, 80, 4), (F16, 16, 64, 2)])
def test_page_calls_step_by_step(ctx, kv, pt, D, skew):
    """Every call once, on pages of 16-, 4- and 2-byte copies (skew: pools off a 16-byte boundary)."""
    p = Pair(ctx, kv=kv, pt=pt, D=D, pages=60, rows=9, max_pages=16, skew=skew, seed=pt)
    p.do("grow", [3, 0, 5], [2 * pt + 1, pt, 1])
    p.same()
    p.do("fork", [3, 3, 0, 8], [1, 2, 7, 6])  # a partly filled row twice, a full one, an empty one
    p.same()
    p.do("fork", [3, 5], [6, 8], deep=True)
    p.same()
    p.do("free", [3, 2, 0], [pt + (pt > 1), 0, 99])
    p.same()
    p.do("grow", [3, 1], [1, 3 * pt])  # row 3 may stand on a shared page
    p.same()
    p.do("free", [7, 5])
    p.same()
    p.do("compact")
    p.same()
    p.do("compact")  # nothing left to move
    p.same()


@pytest.mark.parametrize("seed", range(4))
def test_random_calls(ctx, seed):
    rng = np.random.default_rng(seed)
    pt = int(rng.integers(1, 9))
    p = Pair(ctx, layers=1, pages=int(rng.integers(20, 90)), pt=pt, rows=24, max_pages=10, kvh=1, D=8, seed=seed)
    seen = 0
    for step in range(60):
        op = rng.choice(["grow", "grow", "fork", "fork", "free", "compact"])
        n = int(rng.integers(1, 6))
        rows = [int(r) for r in rng.permutation(24)[:n]]
        if op == "grow":
            p.do(op, rows, [int(a) for a in rng.integers(0, 3 * pt, n)])
        elif op == "fork":
            empty = [r for r in range(24) if p.m.n_kv[r] == 0] or rows
            dst = empty[:n]
            src = [r for r in range(24) if r not in dst]
            p.do(op, [int(s) for s in rng.choice(src, len(dst))], dst, deep=bool(rng.integers(2)))
        elif op == "free":
            p.do(op, rows, None if rng.integers(2) else [int(a) for a in rng.integers(0, 5 * pt, n)])
        else:
            p.do(op)
        seen |= p.m.status
        p.same(pools=step % 10 == 9)
    p.same()
    assert seen & (FULL | TAKEN | LONG)


def test_calls_that_cannot_be_done_have_no_effect(ctx):
    p = Pair(ctx, pages=10, pt=4, rows=6, max_pages=6)
    p.do("grow", [0, 1], [21, 9])  # 6 and 3 pages: one page left
    p.same()
    p.do("grow", [2, 3], [4, 1])
    assert p.m.status == FULL
    p.same()
    p.do("grow", [2, 0], [1, 4])  # row 0 past its table
    assert p.m.status == LONG
    p.same()
    p.do("fork", [0, 1], [2, 3])  # two copies, one page
    assert p.m.status == FULL
    p.same()
    p.do("fork", [1], [0])
    assert p.m.status == TAKEN
    p.same()
    p.do("fork", [1], [3], deep=True)
    assert p.m.status == FULL
    p.same()
    p.do("grow", [2, 1], [0xFFFFFFFF, 1])  # a length past 32 bits
    assert p.m.status == LONG
    p.same()
    p.do("grow", [5, 0], [0, 0])
    p.same()


def test_holes_and_shared_pages(ctx):
    p = Pair(ctx, pages=30, pt=4, rows=6, max_pages=6)
    p.do("grow", [0, 1], [18, 15])
    for s, j in ((0, 1), (0, 4), (1, 3)):  # a page given up in the middle, and a partly filled last one
        p.m.refs[p.m.tables[s][j]] -= 1
        p.m.tables[s][j] = NO_PAGE if j != 3 else 30
    p.put()
    p.do("fork", [0, 1], [2, 3])
    p.same()
    p.do("fork", [0, 1], [4, 5], deep=True)
    p.same()
    p.do("grow", [0, 1], [3, 6])
    p.same()
    p.do("free", [0, 4], [3, 0])
    p.do("compact")
    p.same()


def test_both_rows_of_a_shared_last_page_grow_at_once(ctx):
    p = Pair(ctx, pages=20, pt=8, rows=4, max_pages=4)
    p.do("grow", [0], [16])
    p.do("fork", [0, 0], [1, 2])
    p.do("free", [0, 1, 2], [12, 12, 12])
    p.do("grow", [0, 1], [1, 1])
    p.same()
    p.do("grow", [2], [1])  # alone on the page now
    p.same()


def test_the_longest_lists(ctx):
    n = 1024
    p = Pair(ctx, layers=1, pages=5000, pt=2, kvh=1, D=4, rows=2 * n, max_pages=3)
    p.do("grow", list(range(n)), [1 + i % 5 for i in range(n)])
    p.do("fork", [i // 2 for i in range(n)], list(range(n, 2 * n)))
    p.do("free", list(range(0, 2 * n, 2)))
    p.same()
    p.do("compact")
    p.same()
    with pytest.raises(BadArgument):
        p.c.free(list(range(n + 1)))


def test_a_large_pool(ctx):
    """More pages than one sweep of the plan reads (16 384), the free ones at the far end."""
    p = Pair(ctx, layers=1, pages=40003, pt=1, kvh=1, D=2, rows=4, max_pages=39000)
    p.do("grow", [0, 1], [16380, 20000])
    p.do("grow", [2], [3000])
    p.same()
    p.do("free", [0, 1], [10, 19000])
    p.do("fork", [2], [3], deep=True)
    p.do("compact")
    p.same()


def test_compaction_into_other_tables_leaves_the_old_ones_readable(ctx):
    p = Pair(ctx, pages=40, pt=4, rows=6, max_pages=6)
    p.do("grow", [0, 1, 2, 3], [20, 9, 24, 7])
    p.do("free", [0, 2], [3, 0])
    was_t, was_r = [list(r) for r in p.m.tables], list(p.m.refs)
    t, r, n = (ctx.alloc_n(np.uint32, k) for k in (36, 40, 1))
    p.c.compact(tables_out=t, refs_out=r, n_live=n)
    before = [p.m.row_bits(s) for s in range(6)]
    live = p.m.compact()
    assert ctx.download(n, np.uint32, 1)[0] == live
    assert ctx.download(t, np.uint32, 36).reshape(6, 6).tolist() == p.m.tables
    assert ctx.download(r, np.uint32, 40).tolist() == p.m.refs
    assert ctx.download(p.c.tables, np.uint32, 36).reshape(6, 6).tolist() == was_t
    assert ctx.download(p.c.refs, np.uint32, 40).tolist() == was_r
    assert np.array_equal(ctx.download(p.c.k_pages[1], np.uint16, p.m.k[1].size), p.m.k[1].ravel())
    p.m.tables = was_t
    assert [p.m.row_bits(s) for s in range(6)] == before


# ---- attention ---------------------------------------------------------------------------------

def batch(ctx, lens, H, kvh, D, kv, pt, *, seed=0, begin=None, sinks=False, new=False, pad=0, rows=None, skew=0, holes=(), fill=None, scale=None):
    """One attention call on rows of the given lengths, against the model. Returns the output."""
    rng = np.random.default_rng(seed)
    n_rows = max(len(lens), max(rows) + 1 if rows else 0)
    per = max(1, max(-(-n // pt) for n in lens))
    pages = sum(-(-n // pt) for n in lens) + 4
    p = Pair(ctx, layers=1, pages=pages, pt=pt, kvh=kvh, D=D, kv=kv, rows=n_rows, max_pages=per + 1, n_heads=H, seed=seed, skew=skew)
    ids = [int(x) for x in rng.permutation(pages)]
    at = rows if rows is not None else list(range(len(lens)))
    for s, n in zip(at, lens):
        for j in range(-(-n // pt)):
            p.m.tables[s][j] = ids.pop()
            p.m.refs[p.m.tables[s][j]] = 1
        p.m.n_kv[s] = n
    for s, j in holes:
        p.m.tables[s][j] = NO_PAGE if j % 2 else pages + j
    if fill is not None:  # everything outside the live keys
        live = np.zeros((pages, pt), bool)
        for i, s in enumerate(at):
            for j in range(0 if begin is None else begin[i], lens[i]):
                if p.m.tables[s][j // pt] < pages:
                    live[p.m.tables[s][j // pt], j % pt] = True
        for pool, dev in ((p.m.k, p.c.k_pages), (p.m.v, p.c.v_pages)):
            pool[0][~live] = store(np.array([fill]), kv)[0]
            ctx.upload(dev[0], pool[0])
    p.put()
    n = len(lens)
    width = (H + 2 * kvh) * D + pad
    x = rng.standard_normal((n, width), np.float32)
    q, kn, vn = x[:, :H * D], x[:, H * D:(H + kvh) * D], x[:, (H + kvh) * D:(H + 2 * kvh) * D]
    sk = rng.standard_normal(H, np.float32) if sinks else None
    dx, out = ctx.upload_new(x), ctx.upload_new(np.full(n * H * D + 8, 7.5, np.float32))
    usual, scale = scale is None, D ** -0.5 if scale is None else scale
    kw = dict(q_stride=width, new_stride=width, seqs=rows, kv_begin=None if begin is None else ctx.upload_new(np.array(begin, np.uint32)),
              sinks=None if sk is None else ctx.upload_new(sk))
    if new:
        kw.update(k_new=dx.view(4 * H * D, dx.nbytes - 4 * H * D), v_new=dx.view(4 * (H + kvh) * D, dx.nbytes - 4 * (H + kvh) * D))
    p.c.attn_decode(0, out, dx, n, H, scale, **kw)
    got = ctx.download(out, np.float32, n * H * D + 8)
    assert (got[n * H * D:] == 7.5).all()
    got = got[: n * H * D].reshape(n, H, D)
    want, vmax, amax = attend(p.m, 0, q.reshape(n, H, D), scale, at, begin, sk, kn.reshape(n, kvh, D) if new else None,
                              vn.reshape(n, kvh, D) if new else None)
    tol = attend_tolerance(vmax, amax, D, max(lens))
    err = float(np.abs(got - want).max()) if n else 0.0
    rel = err and float(np.linalg.norm(got - want) / np.linalg.norm(want))
    print(f"attention {lens if len(lens) < 6 else len(lens)} {H}/{kvh} x {D} kv {kv}: max error {err:.2e} (bound {tol:.2e}), relative 2-norm {rel:.2e}")
    assert err <= tol
    if usual:  # scores up to about 5, rounded (D + 8) times at random (5 sqrt(D + 8) EPS each, twice); exp and splits 2^-21
        assert rel <= 2 * 5 * (D + 8) ** 0.5 * EPS + 2.0 ** -21
    for dev, host in ((p.c.k_pages, p.m.k), (p.c.v_pages, p.m.v)):  # the new tokens stored, nothing else written
        assert np.array_equal(ctx.download(dev[0], host.dtype, host[0].size), host[0].ravel())
    p.c.attn_decode(0, out, dx, n, H, scale, **kw)  # the same bits again
    assert np.array_equal(ctx.download(out, np.float32, n * H * D).reshape(n, H, D), got)
    return got


SHAPES = [(64, 8, 64), (32, 4, 128), (20, 5, 80), (12, 2, 96), (16, 1, 256), (7, 7, 72), (4, 4, 8), (6, 2, 5), (9, 3, 130), (8, 1, 300), (5, 5, 1024)]


@pytest.mark.parametrize("kv", [BF16, F16, F32])
@pytest.mark.parametrize("H, kvh, D", SHAPES)
def test_attention_shapes(ctx, H, kvh, D, kv):
    """Every head layout and cache type on ragged rows: empty, one token, around a tile and a page."""
    batch(ctx, [33, 0, 1, 16, 17, 90, 0, 8, 31], H, kvh, D, kv, 16, seed=D, sinks=D % 2 == 0, new=True, pad=3)


@pytest.mark.parametrize("pt", [1, 3, 16, 17, 64, 200])
def test_attention_page_sizes(ctx, pt):
    batch(ctx, [130, 64, 65, 1], 16, 2, 64, BF16, pt, seed=pt, new=pt != 17)
    batch(ctx, [130, 64, 65, 1], 6, 3, 40, F32, pt, seed=pt, new=pt == 17)


@pytest.mark.parametrize("H, kvh, D, kv", [(8, 8, 64, BF16), (8, 1, 64, F16), (24, 2, 128, BF16), (34, 2, 64, BF16), (11, 11, 64, F16), (13, 1, 32, F32)])
def test_attention_splits(ctx, H, kvh, D, kv):
    """Long and short rows together: rows in one CTA, rows over many, and several rows a CTA; groups
    larger than a tensor-core tile's heads, and fewer heads than warps."""
    batch(ctx, [3000, 5, 0, 1700, 200, 40, 1], H, kvh, D, kv, 32, seed=H, sinks=True, new=True)
    batch(ctx, [20] * 700, H, kvh, D, kv, 32, seed=H)


def test_attention_of_one_long_row(ctx):
    batch(ctx, [20011], 8, 1, 128, BF16, 64, seed=1, new=True)
    batch(ctx, [9001], 4, 2, 80, F32, 64, seed=2)


@pytest.mark.parametrize("D", [40, 48, 56, 72, 80, 88, 96, 104, 112, 120, 136, 248])
@pytest.mark.parametrize("kv", [BF16, F16])
def test_attention_between_the_usual_head_sizes(ctx, D, kv):
    """16-bit heads of every multiple of 8 around the tensor-core tiles' sizes: rows of several tiles,
    pages that end inside one, windows, and a pool that is NaN everywhere outside the live keys."""
    lens, begin = [700, 0, 129, 128, 5, 390, 1], [3, 0, 0, 127, 5, 257, 0]
    batch(ctx, lens, 15, 3, D, kv, 7, seed=D, sinks=True, new=D % 16 == 0, pad=D % 3)
    batch(ctx, lens, 20, 2, D, kv, 24, seed=D, begin=begin, fill=np.nan)


@pytest.mark.parametrize("H, kvh, D", [(5, 5, 36), (8, 8, 64), (20, 5, 76), (14, 7, 80), (6, 2, 84), (24, 3, 128), (4, 1, 132), (16, 2, 252), (3, 3, 256)])
def test_f32_attention_on_the_tensor_cores(ctx, H, kvh, D):
    """f32 heads around the tiles' sizes: long and short rows together, one computing warp to eight with
    their loading warps, pages that end inside a tile, windows, NaN outside the live keys, many rows."""
    lens = [1300, 0, 129, 16, 5, 390, 1]
    batch(ctx, lens, H, kvh, D, F32, 7, seed=D, sinks=True, new=True, pad=D % 3)
    batch(ctx, lens, H, kvh, D, F32, 16, seed=D, begin=[3, 0, 0, 15, 5, 257, 0], fill=np.nan)
    batch(ctx, [9] * 900, H, kvh, D, F32, 16, seed=D, new=True)


def test_attention_windows(ctx):
    lens = [100, 40, 3, 7, 90, 12]
    batch(ctx, lens, 8, 2, 64, BF16, 16, begin=[70, 0, 2, 7, 89, 30], sinks=True, new=True)  # row 3 has nothing left, row 5's start is past its end
    batch(ctx, lens, 8, 2, 48, F32, 16, begin=[70, 0, 2, 7, 89, 30], new=True)


@pytest.mark.parametrize("kv, D", [(BF16, 64), (F16, 128), (F32, 64), (BF16, 24)])
@pytest.mark.parametrize("fill", [np.nan, np.inf, -np.inf, np.finfo(np.float32).min])
def test_what_lies_outside_the_row_does_not_matter(ctx, kv, D, fill):
    """NaN, infinities and the lowest value in holes, behind the last token and before the window."""
    with np.errstate(over="ignore"):
        batch(ctx, [50, 33, 20], 8, 2, D, kv, 8, begin=[3, 0, 10], holes=[(0, 2), (1, 1)], fill=fill, sinks=True, new=True)


def test_a_row_of_holes_is_zero(ctx):
    for kv, D in ((BF16, 64), (F32, 20)):
        got = batch(ctx, [30, 16, 9], 4, 2, D, kv, 8, holes=[(1, 0), (1, 1), (0, 3)], sinks=True, new=True)
        assert (got[1] == 0).all()


def test_rows_by_list(ctx):
    batch(ctx, [33, 5, 0, 70], 8, 2, 64, BF16, 16, rows=[6, 1, 9, 3], new=True)
    batch(ctx, [33], 8, 2, 64, F32, 16, rows=[4])


@pytest.mark.parametrize("skew", [2, 4, 8])
def test_pools_off_a_16_byte_boundary(ctx, skew):
    batch(ctx, [40, 9], 8, 2, 64, F16, 16, skew=skew, new=True)
    if skew >= 4:
        batch(ctx, [40, 9], 8, 2, 64, F32, 16, skew=skew, new=True)


@pytest.mark.parametrize("kv", [BF16, F16, F32])
def test_large_and_tiny_queries(ctx, kv):
    """Scores from nearly uniform to nearly one-hot; the bound grows with them."""
    for scale in (1e-6, 1.0, 6.0, -0.5):
        batch(ctx, [70, 300], 8, 2, 64, kv, 16, scale=scale, sinks=True)


def test_accuracy_over_a_long_row(ctx):
    """The 2-norm error of a 30 000-key row stays at f32's level: the sums over the keys do not drift."""
    rng = np.random.default_rng(5)
    H, kvh, D, n, pt = 8, 1, 128, 30000, 64
    for kv in (BF16, F16):
        p = Pair(ctx, layers=1, pages=-(-n // pt), pt=pt, kvh=kvh, D=D, kv=kv, rows=1, max_pages=-(-n // pt), n_heads=H)
        p.do("grow", [0], [n])
        q = rng.standard_normal((1, H, D)).astype(np.float32)
        out = ctx.alloc_n(np.float32, H * D)
        p.c.attn_decode(0, out, ctx.upload_new(q), 1, H, D ** -0.5)
        want, _, _ = attend(p.m, 0, q, D ** -0.5)
        rel = np.linalg.norm(ctx.download(out, np.float32, H * D).reshape(want.shape) - want) / np.linalg.norm(want)
        print(f"kv {kv}: relative 2-norm error {rel:.2e}")
        # scores of magnitude ~4 rounded (D + 8) times at random: ~ 4 sqrt(D) EPS each, twice; exp 2^-22
        assert rel <= 2 * 4 * D ** 0.5 * EPS + 2.0 ** -21


@pytest.mark.parametrize("kv, kvh, D", [(BF16, 4, 64), (BF16, 4, 80), (F32, 4, 64), (F16, 8, 128), (F32, 3, 200)])
def test_one_workspace_serves_any_number_of_heads(ctx, kv, kvh, D):
    """A cache made for many query heads, then read with fewer, whose work may be cut more finely."""
    p = Pair(ctx, layers=1, pages=200, pt=16, kvh=kvh, D=D, kv=kv, rows=3, max_pages=80, n_heads=24 * kvh)
    p.do("grow", [0, 1, 2], [1100, 3, 190])
    rng = np.random.default_rng(0)
    for group in (24, 17, 16, 8, 5, 4, 1):
        q = rng.standard_normal((3, group * kvh, D)).astype(np.float32)
        out = ctx.alloc_n(np.float32, q.size)
        p.c.attn_decode(0, out, ctx.upload_new(q), 3, group * kvh, D ** -0.5)
        want, vmax, amax = attend(p.m, 0, q, D ** -0.5)
        assert np.abs(ctx.download(out, np.float32, q.size).reshape(q.shape) - want).max() <= attend_tolerance(vmax, amax, D, 1100)


def test_attention_without_rows_and_its_checks(ctx):
    p = Pair(ctx, n_heads=4)
    b = ctx.alloc(4 * 8 * 4 * 64)
    p.c.attn_decode(0, b, b, 0, 4, 1.0)
    p.c.attn_decode(0, b, b, 8, 4, 1.0)  # every row empty
    assert (ctx.download(b, np.float32, 8 * 4 * 64) == 0).all()
    for kw in (dict(n_heads=5), dict(n_heads=0), dict(n_seq=9), dict(layer=2), dict(n_seq=-1)):
        a = dict(layer=0, n_seq=2, n_heads=4)
        a.update(kw)
        with pytest.raises((BadArgument, BufferTooSmall)):
            p.c.attn_decode(a["layer"], b, b, a["n_seq"], a["n_heads"], 1.0)
    with pytest.raises(BufferTooSmall):
        p.c.attn_decode(0, b.view(0, 1000), b, 2, 4, 1.0)
    with pytest.raises(BadArgument):
        p.c.attn_decode(0, b, b, 2, 4, 1.0, k_new=b, v_new=b, seqs=[1, 1])
    with pytest.raises(Exception):
        p.c.attn_decode(0, b, b, 2, 4, 1.0, k_new=b)


# ---- together, as a serving loop uses them -------------------------------------------------------

def step_inputs(rng, n, H, kvh, D):
    return (rng.standard_normal((n, H, D), np.float32), rng.standard_normal((n, kvh, D), np.float32), rng.standard_normal((n, kvh, D), np.float32))


@pytest.mark.parametrize("kv, H, kvh, D, pt", [(BF16, 16, 2, 64, 8), (F16, 8, 2, 128, 5), (F32, 6, 3, 40, 4)])
def test_a_serving_loop(ctx, kv, H, kvh, D, pt):
    """Rows are started, decoded over two layers, scored, forked from the better and dropped from the
    worse, cut back and compacted; every step's attention, pools and tables follow the model."""
    rng = np.random.default_rng(D)
    p = Pair(ctx, layers=2, pages=120, pt=pt, kvh=kvh, D=D, kv=kv, rows=10, max_pages=14, n_heads=H, seed=D)
    p.do("grow", [0, 1, 2], [13, 1, 2 * pt])  # prompts, whose keys the pools hold already
    alive, V = [0, 1, 2], 500
    for step in range(8):
        p.do("grow", alive, [1] * len(alive))
        n = len(alive)
        for layer in range(2):
            q, kn, vn = step_inputs(rng, n, H, kvh, D)
            out = ctx.alloc_n(np.float32, n * H * D)
            p.c.attn_decode(layer, out, ctx.upload_new(q), n, H, D ** -0.5, seqs=alive, k_new=ctx.upload_new(kn), v_new=ctx.upload_new(vn))
            want, vmax, amax = attend(p.m, layer, q, D ** -0.5, alive, k_new=kn, v_new=vn)
            got = ctx.download(out, np.float32, n * H * D).reshape(want.shape)
            assert np.abs(got - want).max() <= attend_tolerance(vmax, amax, D, max(p.m.n_kv))
        p.same()
        logits = rng.standard_normal((n, V)).astype(np.float32) + got.reshape(n, -1)[:, :1]
        ids, top = ctx.alloc_n(np.uint32, n * 2), ctx.alloc_n(np.float32, n * 2)
        ctx.token_logprobs(ctx.upload_new(logits), F32, n, V, k=2, top_ids=ids, top_logprobs=top)
        assert (ctx.download(ids, np.uint32, 2 * n).reshape(n, 2)[:, 0] == logits.argmax(1)).all()
        order = np.argsort(-ctx.download(top, np.float32, 2 * n).reshape(n, 2)[:, 0])
        best, worst = alive[order[0]], alive[order[-1]]
        if len(alive) > 2:
            p.do("free", [worst])
            alive.remove(worst)
        new = [r for r in range(10) if p.m.n_kv[r] == 0][:2]
        p.do("fork", [best] * len(new), new, deep=step == 3)
        alive += new
        if step % 3 == 2:
            p.do("free", [alive[0]], [max(1, p.m.n_kv[alive[0]] - pt - 1)])  # rejected tokens
            p.do("compact")
        p.same()


def test_a_captured_step_follows_the_cache(ctx):
    """Growing, attention and scores captured once: each replay takes the lengths and tables it finds."""
    torch = pytest.importorskip("torch")
    H, kvh, D, pt, n, V = 8, 2, 64, 4, 3, 300
    rng = np.random.default_rng(3)
    p = Pair(ctx, layers=1, pages=40, pt=pt, kvh=kvh, D=D, rows=4, max_pages=12, n_heads=H)
    p.do("grow", [0, 1, 3], [5, 1, 9])
    q, kn, vn = step_inputs(rng, n, H, kvh, D)
    dq, dk, dv, out = ctx.upload_new(q), ctx.upload_new(kn), ctx.upload_new(vn), ctx.alloc_n(np.float32, n * H * D)
    logits, ent = ctx.upload_new(rng.standard_normal((n, V), np.float32)), ctx.alloc_n(np.float32, n)

    def step():
        p.c.grow([0, 1, 3], [1, 1, 1])
        p.c.attn_decode(0, out, dq, n, H, 0.125, seqs=[0, 1, 3], k_new=dk, v_new=dv)
        ctx.token_logprobs(logits, F32, n, V, entropy=ent)

    def check():
        p.m.grow([0, 1, 3], [1, 1, 1])
        want, vmax, amax = attend(p.m, 0, q, 0.125, [0, 1, 3], k_new=kn, v_new=vn)
        got = ctx.download(out, np.float32, n * H * D).reshape(want.shape)
        assert np.abs(got - want).max() <= attend_tolerance(vmax, amax, D, 50)
        assert np.isfinite(ctx.download(ent, np.float32, n)).all()
        p.same()

    step()  # attributes are set on the first call, outside a capture
    check()
    stream = torch.cuda.ExternalStream(ctx.lib.moearc_x_stream(ctx.raw))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    for _ in range(6):
        with torch.cuda.stream(stream):
            graph.replay()
        ctx.sync()
        check()
    p.do("free", [1])
    p.do("fork", [3], [1])
    p.do("compact")
    with torch.cuda.stream(stream):
        graph.replay()
    check()
    del graph


def test_two_contexts_at_once():
    """Two caches on two streams, interleaved without waiting: neither sees the other."""
    a, b = Context(), Context()
    H, kvh, D, n = 16, 2, 128, 4
    rng = np.random.default_rng(9)
    sides = []
    for c, kv in ((a, BF16), (b, F16)):
        p = Pair(c, layers=1, pages=400, pt=16, kvh=kvh, D=D, kv=kv, rows=n, max_pages=90, n_heads=H, seed=kv)
        p.do("grow", list(range(n)), [1200, 7, 300, 64])
        q = rng.standard_normal((n, H, D)).astype(np.float32)
        sides.append((p, q, c.upload_new(q), [c.alloc_n(np.float32, n * H * D) for _ in range(20)]))
    for i in range(20):
        for p, q, dq, outs in sides:
            p.c.attn_decode(0, outs[i], dq, n, H, D ** -0.5)
    for p, q, dq, outs in sides:
        want, vmax, amax = attend(p.m, 0, q, D ** -0.5)
        first = p.ctx.download(outs[0], np.float32, want.size)
        assert np.abs(first.reshape(want.shape) - want).max() <= attend_tolerance(vmax, amax, D, 1200)
        for o in outs[1:]:
            assert np.array_equal(p.ctx.download(o, np.float32, want.size), first)
    for c in (a, b):
        c.close()


@pytest.mark.parametrize("kv, H, kvh, D, pt", [(BF16, 16, 4, 128, 16), (F32, 8, 4, 128, 16)])
def test_pools_past_32_bit_offsets(ctx, kv, H, kvh, D, pt):
    """Pages beyond 4 GiB (and 2^31 elements) of a pool: attention, the new token's store and copies."""
    size = 4 if kv == F32 else 2
    page_bytes = pt * kvh * D * size
    pages = (5 << 30) // page_bytes + 5
    small = Paged(1, 8, pt, kvh, D, kv, 3, 6, seed=4)
    far = [pages - 1 - i for i in range(4)] + list(range(4))  # where the model's pages lie
    pools = [ctx.alloc(pages * page_bytes) for _ in range(2)]
    for pool, host in zip(pools, (small.k, small.v)):
        for i, f in enumerate(far):
            ctx.upload(pool.view(f * page_bytes, page_bytes), host[0, i])
    c = KvCache(ctx, n_layer=1, n_pages=pages, page_tokens=pt, n_kv_heads=kvh, head_dim=D, kv_type=kv, max_seq=3, max_pages=6,
                n_heads=H, k_pages=[pools[0]], v_pages=[pools[1]])
    small.tables[0][:3], small.n_kv[0] = [0, 4, 1], 3 * pt - 2
    refs = np.zeros(pages, np.uint32)
    refs[:4] = 1  # taken, so that the copies below go to pages that are far, then near
    refs[far[0]] = refs[far[1]] = 1
    tables = np.full((3, 6), NO_PAGE, np.uint32)
    tables[0, :3] = [far[p] for p in small.tables[0][:3]]
    ctx.upload(c.tables, tables)
    ctx.upload(c.n_kv, np.array(small.n_kv, np.uint32))
    ctx.upload(c.refs, refs)
    rng = np.random.default_rng(1)
    q, kn, vn = step_inputs(rng, 1, H, kvh, D)
    out = ctx.alloc_n(np.float32, H * D)
    c.attn_decode(0, out, ctx.upload_new(q), 1, H, D ** -0.5, k_new=ctx.upload_new(kn), v_new=ctx.upload_new(vn))
    want, vmax, amax = attend(small, 0, q, D ** -0.5, k_new=kn, v_new=vn)
    assert np.abs(ctx.download(out, np.float32, H * D).reshape(want.shape) - want).max() <= attend_tolerance(vmax, amax, D, 3 * pt)
    for pool, host in zip(pools, (small.k, small.v)):
        for i, f in enumerate(far):
            assert np.array_equal(ctx.download(pool.view(f * page_bytes, page_bytes), host.dtype, host[0, i].size), host[0, i].ravel())
    c.fork([0], [1], deep=True)
    t = ctx.download(c.tables, np.uint32, 18).reshape(3, 6)
    assert t[1, :3].tolist() == [4, 5, 6] and c.status() == 0
    refs[:] = 1  # only far pages are free
    refs[far[2]] = refs[far[3]] = 0
    ctx.upload(c.refs, refs)
    c.fork([0], [2])
    t = ctx.download(c.tables, np.uint32, 18).reshape(3, 6)
    assert t[2, :3].tolist() == [t[0, 0], t[0, 1], min(far[2], far[3])]
    for a, b in zip(list(t[0, :3]) * 2, list(t[1, :3]) + list(t[2, :3])):
        for pool in pools:
            x, y = (ctx.download(pool.view(int(f) * page_bytes, page_bytes), np.uint32, page_bytes // 4) for f in (a, b))
            assert np.array_equal(x, y)
    for b in pools:
        b.free()

"""Token log probabilities on the B200 against 64-bit arithmetic: values within bounds derived from
the roundings, alternatives exactly (value, then lowest id)."""
import numpy as np
import pytest

from moearc_b200 import BadArgument, BufferTooSmall, Context
from paged_model import BF16, EPS, F16, F32, store

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = Context()
    yield c
    c.close()


def as_f32(bits, ty):
    if ty == F32:
        return bits.view(np.float32)
    return bits.view(np.float16).astype(np.float32) if ty == F16 else (bits.astype(np.uint32) << 16).view(np.float32)


def check(ctx, x, ty, k=0, stride=None, scale=1.0, tokens=None, offset=0, only=None):
    """One call on rows x (f32, rounded to the type) against 64 bits."""
    n, V = x.shape
    stride = stride or V
    with np.errstate(over="ignore"):
        bits = store(np.full((n, stride), 1e30 if ty != F16 else 6e4, np.float32), ty).reshape(n, stride)
        bits[:, :V] = store(x, ty).reshape(n, V)
    size = bits.itemsize
    buf = ctx.alloc(bits.nbytes + offset * size)
    ctx.upload(buf.view(offset * size, bits.nbytes), bits)
    tokens = np.random.default_rng(n + V).integers(0, V, n) if tokens is None else np.asarray(tokens)
    lp, ent = ctx.upload_new(np.full(n + 1, 9.0, np.float32)), ctx.upload_new(np.full(n + 1, 9.0, np.float32))
    ids, top = ctx.upload_new(np.full(n * k + 1, 77, np.uint32)), ctx.upload_new(np.full(n * k + 1, 9.0, np.float32))
    kw = dict(tokens=ctx.upload_new(tokens.astype(np.uint32)), logprob=lp) if only != "entropy" else {}
    if only != "logprob":
        kw["entropy"] = ent
    if k:
        kw.update(k=k, top_ids=ids, top_logprobs=top)
    ctx.token_logprobs(buf.view(offset * size, bits.nbytes), ty, n, V, row_stride=stride, scale=scale, **kw)
    g_lp, g_ent = ctx.download(lp, np.float32, n + 1), ctx.download(ent, np.float32, n + 1)
    g_ids, g_top = ctx.download(ids, np.uint32, n * k + 1), ctx.download(top, np.float32, n * k + 1)
    assert g_lp[n] == 9.0 and g_ent[n] == 9.0 and g_ids[n * k] == 77 and g_top[n * k] == 9.0
    y32 = as_f32(bits[:, :V], ty) * np.float32(scale)
    y = y32.astype(np.float64)
    for r in range(n):
        M = y[r].max()
        if M == -np.inf:
            if only != "entropy":
                assert g_lp[r] == (-np.inf if tokens[r] < V else 0.0)
            assert only == "logprob" or g_ent[r] == 0.0
            want = np.full(V, -np.inf)
            tol = 0.0
        else:
            e = np.exp(y[r] - M)
            L = e.sum()
            want = y[r] - M - np.log(L)
            S = float((e * np.where(e > 0, y[r] - M, 0.0)).sum()) / L
            # each weight: its exponent rounded twice where |d| e^d <= 1/e, the exponential 2^-22; V / 256
            # sums a thread and a tree of joins, whose factors are exponentials too; log one rounding of itself
            rel = 2.0 ** -21 + 2 * EPS + (V / 256 + 64) * EPS + 12 * 2.0 ** -21
            fin = np.abs(np.where(np.isfinite(want), y[r], 0.0))
            tol = rel + EPS * (2 * fin.max() + 2 * abs(M) + 4 * abs(np.log(L)) + 2)
            if only != "entropy":
                if tokens[r] >= V:
                    assert g_lp[r] == 0.0
                elif np.isfinite(want[tokens[r]]):
                    assert abs(g_lp[r] - want[tokens[r]]) <= tol
                else:
                    assert g_lp[r] == -np.inf
            if only != "logprob":
                H = np.log(L) - S
                assert abs(g_ent[r] - H) <= tol + 2 * rel * (abs(S) + 1), (g_ent[r], H)
        if k:
            order = np.lexsort((np.arange(V), -y32[r].astype(np.float64)))[:k]
            assert g_ids[r * k:(r + 1) * k].tolist() == order.tolist()
            g, w = g_top[r * k:(r + 1) * k], want[order]
            assert ((g == w) | (np.abs(np.where(np.isfinite(w), g - w, 0.0)) <= tol) & np.isfinite(w)).all()


@pytest.mark.parametrize("ty", [F32, F16, BF16])
@pytest.mark.parametrize("V", [1, 2, 31, 255, 1000, 4099, 40001])
@pytest.mark.parametrize("n", [1, 5])
def test_sizes_and_types(ctx, n, V, ty):
    x = np.random.default_rng(V).standard_normal((n, V)).astype(np.float32) * 3
    check(ctx, x, ty, k=min(V, 32))
    check(ctx, x, ty, k=min(V, 5), stride=V + 3, offset=1, scale=0.7)  # rows on every alignment
    check(ctx, x, ty)


@pytest.mark.parametrize("n, V", [(1, 200003), (3, 131072), (40, 50001), (700, 3001), (1500, 2003)])
def test_every_cluster_size(ctx, n, V):
    x = np.random.default_rng(n).standard_normal((n, V)).astype(np.float32) * 2
    check(ctx, x, F32, k=20)
    check(ctx, x, BF16, k=7)


@pytest.mark.parametrize("k", [1, 2, 8, 9, 32])
def test_equal_values_go_to_the_lowest_id(ctx, k):
    """Ties over a whole row, so that the list of candidates overflows many times, and in steps."""
    for V in (100, 3000, 60000):
        check(ctx, np.zeros((2, V), np.float32), F32, k=k)
        check(ctx, np.floor(np.arange(V, dtype=np.float32) / 700)[None], F32, k=k)
        check(ctx, -np.floor(np.arange(V, dtype=np.float32) / 700)[None], BF16, k=k)
        x = np.zeros((1, V), np.float32)
        x[0, ::2] = -0.0
        check(ctx, x, F32, k=k)
        check(ctx, np.arange(V, dtype=np.float32)[None] * 1e-3, F32, k=k)  # ascending


def test_masked_rows(ctx):
    rng = np.random.default_rng(0)
    x = rng.standard_normal((6, 5000)).astype(np.float32)
    x[0] = -np.inf
    x[1, 17:] = -np.inf
    x[2, :4999] = -np.inf
    x[3, rng.random(5000) < 0.99] = -np.inf
    x[4, 100:3000] = np.finfo(np.float32).min
    check(ctx, x, F32, k=20)
    check(ctx, x, F32, k=20, tokens=[3, 4000, 10, 0, 200, 5000])
    check(ctx, x[:4], BF16, k=20)
    check(ctx, x, F32, k=20, only="entropy")
    check(ctx, x, F32, only="logprob")


def test_wide_values(ctx):
    rng = np.random.default_rng(1)
    x = rng.standard_normal((3, 3000)).astype(np.float32)
    x[0] *= 1e4
    x[1] += 3e4
    x[2, 5] = 200.0
    check(ctx, x, F32, k=6)
    check(ctx, x, F32, k=6, scale=1e-3)


def test_nan_and_infinity_are_seen(ctx):
    x = np.random.default_rng(2).standard_normal((3, 3000)).astype(np.float32)
    x[0, 2000] = np.nan
    x[1, 7] = np.inf
    x[1, 9] = 1.0
    ids, top, lp, ent = ctx.alloc_n(np.uint32, 12), ctx.alloc_n(np.float32, 12), ctx.alloc_n(np.float32, 3), ctx.alloc_n(np.float32, 3)
    ctx.token_logprobs(ctx.upload_new(x), F32, 3, 3000, tokens=ctx.upload_new(np.array([1, 7, 3], np.uint32)), logprob=lp, entropy=ent, k=4, top_ids=ids, top_logprobs=top)
    lp, ent, top = ctx.download(lp, np.float32, 3), ctx.download(ent, np.float32, 3), ctx.download(top, np.float32, 12).reshape(3, 4)
    assert np.isnan(lp[:2]).all() and np.isnan(ent[:2]).all() and np.isnan(top[:2]).all()
    assert np.isfinite(lp[2]) and np.isfinite(ent[2]) and np.isfinite(top[2]).all()
    ids = ctx.download(ids, np.uint32, 12).reshape(3, 4)
    assert ids[0].tolist() == [i for i in np.lexsort((np.arange(3000), -np.where(np.isnan(x[0]), -np.inf, x[0]).astype(np.float64)))[:4]]
    assert ids[1, 0] == 7


def test_checks(ctx):
    b = ctx.alloc(400)
    with pytest.raises(BufferTooSmall):
        ctx.token_logprobs(b, F32, 2, 100, entropy=b)
    with pytest.raises(BufferTooSmall):
        ctx.token_logprobs(b, F32, 1, 100, k=101, top_ids=b, top_logprobs=b)
    with pytest.raises(BadArgument):
        ctx.token_logprobs(b, F32, 1, 100, k=33, top_ids=b, top_logprobs=b)
    with pytest.raises(BadArgument):
        ctx.token_logprobs(b, 39, 1, 100, entropy=b)
    ctx.token_logprobs(b, F32, 0, 100, entropy=b)


def test_rows_past_32_bit_offsets(ctx):
    """The last row of logits starts beyond 2^32 elements."""
    V, n = 200003, 22000
    buf = ctx.alloc(n * V * 2)
    x = np.random.default_rng(7).standard_normal(V).astype(np.float32)
    bits = store(x, BF16)
    ctx.upload(buf.view((n - 1) * V * 2, V * 2), bits)
    ids, top, ent = ctx.alloc_n(np.uint32, n), ctx.alloc_n(np.float32, n), ctx.alloc_n(np.float32, n)
    ctx.token_logprobs(buf, BF16, n, V, entropy=ent, k=1, top_ids=ids, top_logprobs=top)
    y = as_f32(bits, BF16).astype(np.float64)
    assert ctx.download(ids, np.uint32, n)[-1] == int(y.argmax())
    lse = np.log(np.exp(y - y.max()).sum()) + y.max()
    assert abs(ctx.download(top, np.float32, n)[-1] - (y.max() - lse)) <= 1e-4  # as in check(): V / 256 sums
    buf.free()

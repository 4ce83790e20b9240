"""Decode attention over the paged cache where single roundings would show: weights many powers of two
below a row's largest, values and weights near the ends of the number range, rows of one key."""
import numpy as np
import pytest

from moearc_b200 import Context
from moearc_b200.kvcache import KvCache
from paged_model import BF16, EPS, F16, F32, Paged, attend, load, store

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = Context()
    yield c
    c.close()


def run(ctx, n, rows, H, kvh, D, kv, q, fill, pt=16):
    """Attention of `rows` rows of n tokens each whose stored keys and values are fill(k, v) of
    normal ones, f32 [rows, n, kvh, D]. Returns (output, the exact one, values as stored)."""
    per = -(-n // pt)
    m = Paged(1, rows * per, pt, kvh, D, kv, rows, per, seed=D)
    m.grow(list(range(rows)), [n] * rows)
    k, v = (load(p[0], kv).astype(np.float32).reshape(rows, per * pt, kvh, D) for p in (m.k, m.v))
    fill(k[:, :n], v[:, :n])
    for p, x in ((m.k, k), (m.v, v)):
        p[0] = store(x, kv).reshape(p[0].shape)
    pools = [[ctx.upload_new(p[0])] for p in (m.k, m.v)]
    c = KvCache(ctx, n_layer=1, n_pages=rows * per, page_tokens=pt, n_kv_heads=kvh, head_dim=D, kv_type=kv, max_seq=rows, max_pages=per,
                n_heads=H, k_pages=pools[0], v_pages=pools[1])
    c.grow(list(range(rows)), [n] * rows)
    out = ctx.alloc_n(np.float32, q.size)
    c.attn_decode(0, out, ctx.upload_new(q), rows, H, D ** -0.5)
    got = ctx.download(out, np.float32, q.size).reshape(q.shape)
    assert c.status() == 0
    return got, attend(m, 0, q, D ** -0.5)[0], load(m.v[0], kv).reshape(rows, per * pt, kvh, D)[:, :n]


def queries(rows, H, D, first=8.0):
    q = np.random.default_rng(D).standard_normal((rows, H, D)).astype(np.float32)
    q[:, :, 0] = first
    return q


SHAPES = [(8, 2, 64), (16, 2, 128), (6, 2, 80), (16, 1, 256), (4, 4, 20), (8, 1, 48)]


@pytest.mark.parametrize("gap", [10, 15, 18, 20, 25, 30])
@pytest.mark.parametrize("kv", [F16, BF16, F32])
def test_weights_far_below_a_key_that_adds_nothing(ctx, kv, gap):
    """One key `gap` above the others in score whose value is zero (an attention sink in the cache): the
    output is the sum of the other weights alone, and keeps its own relative accuracy.

    With X = gap + 6 the largest |score|: the scale's two roundings, the product's, the largest's and the
    difference's are 5 X EPS of a weight (the high key's own product is exact); the others' scores, up to
    5, are rounded (D + 8) times at random, twice; exponential and split 2^-21; the sums over n keys and
    a join at random."""
    for H, kvh, D in SHAPES:
        for n, at in ((300, 0), (3000, 1700)):
            def fill(k, v):
                k[..., 0] = 0
                k[:, at] = 0
                k[:, at, :, 0] = gap / (8.0 * D ** -0.5)
                v[:, at] = 0
            got, want, _ = run(ctx, n, 2, H, kvh, D, kv, queries(2, H, D), fill)
            rel = np.linalg.norm(got - want) / np.linalg.norm(want)
            print(f"kv {kv} {H}/{kvh} x {D}, {n} keys, gap {gap}: relative 2-norm error {rel:.2e}")
            assert rel <= (5 * (gap + 6) + 2 * 5 * (D + 8) ** 0.5 + 5 * (n / 8) ** 0.5) * EPS + 2.0 ** -21


@pytest.mark.parametrize("kv", [BF16, F32])
def test_values_of_large_magnitude(ctx, kv):
    """Values of 2^116 to 2^117 and scores that rise by seven powers of two half way along a row: no
    partial sum leaves the range, as none does in a softmax whose weights are at most one."""
    for H, kvh, D in SHAPES:
        def fill(k, v):
            k[..., 0] = 0
            k[:, 300:, :, 0] = 7.0 * np.log(2) / (8.0 * D ** -0.5)
            k[..., 1:] *= 0.01
            v[...] = (1 + np.abs(v) % 1) * np.float32(2.0 ** 116)
        got, want, v = run(ctx, 600, 100, H, kvh, D, kv, queries(100, H, D), fill)
        assert np.isfinite(got).all()
        # scores up to 5: five roundings of them, D + 8 of their parts; weights and sums as above
        rel = np.abs(got - want).max() / np.abs(v).max()
        print(f"kv {kv} {H}/{kvh} x {D}: error over the largest value {rel:.2e}")
        assert rel <= 2 * (5 * (5 + 5) + 2 * (D + 8) + 600 / 8 + 64) * EPS + 2.0 ** -20


def test_finite_ends_of_the_range_where_they_add_nothing(ctx):
    """The largest finite values in live keys, in a channel where q is zero and behind a weight of zero, and in q
    in a channel where the keys are (f16 caches: 2^10, as their terms of q are a head's fixed-point numbers)."""
    for kv, most in ((F32, np.finfo(np.float32).max), (BF16, np.float32(2.0 ** 128 - 2.0 ** 120)), (F16, np.float32(65504.0))):
        for H, kvh, D in SHAPES:
            q = queries(2, H, D)
            q[:, :, 1] = 0
            q[:, :, 3] = 1024 if kv == F16 else np.finfo(np.float32).max
            q[:, ::2, 3] *= -1

            def fill(k, v):
                k[:, ::3, :, 1] = most
                k[:, 1::3, :, 1] = -most
                k[:, 7, :, 0] = -3000.0
                k[:, 7, :, 2:] = 0
                k[:, :, :, 3] = 0
                v[:, 7] = most
                v[:, 7, :, ::2] = -most
            got, want, _ = run(ctx, 200, 2, H, kvh, D, kv, q, fill)
            assert np.isfinite(got).all(), (kv, H, kvh, D)
            rel = np.linalg.norm(got - want) / np.linalg.norm(want)
            # channel 0 adds 8 N(0, 1) D^-0.5 to the scores: up to 15 in all, five roundings of them
            assert rel <= (5 * 15 + 2 * 5 * (D + 8) ** 0.5 + 25) * EPS + 2.0 ** -21


@pytest.mark.parametrize("kv", [F32, F16, BF16])
def test_a_row_of_one_key_is_its_value(ctx, kv):
    """Its weight is one: the output is the stored value, every bit of it."""
    for H, kvh, D in SHAPES + [(8, 8, 64), (32, 4, 128), (5, 5, 36), (24, 2, 96)]:
        got, _, v = run(ctx, 1, 40, H, kvh, D, kv, queries(40, H, D), lambda k, v: None)
        want = np.repeat(v[:, 0], H // kvh, axis=1).astype(np.float32)
        assert np.array_equal(got, want), (kv, H, kvh, D)

"""Token log probabilities where a scaled logit leaves f32's range: masks of the type's lowest finite value
under a temperature below one, and logits so large that they become infinite."""
import numpy as np
import pytest

from moearc_b200 import Context
from paged_model import BF16, F32
from test_gpu_logprobs import check

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = Context()
    yield c
    c.close()


@pytest.mark.parametrize("V", [40, 5000, 200003])
@pytest.mark.parametrize("ty, least", [(F32, np.finfo(np.float32).min), (BF16, np.float32(2.0 ** 120 - 2.0 ** 128))])
def test_masks_of_the_lowest_value_under_a_scale(ctx, ty, least, V):
    """x = scale logit is -inf there: a row of nothing else has entropy 0 and log probabilities of -inf."""
    x = np.random.default_rng(V).standard_normal((4, V)).astype(np.float32)
    x[0] = least
    x[1, : V // 2] = least
    x[2, 3:] = least
    x[3, ::2] = -np.inf
    x[3, 1::2] = least
    with np.errstate(over="ignore", invalid="ignore"):
        for k in (0, 5):
            check(ctx, x, ty, k=k, scale=1.25)
            check(ctx, x, ty, k=k, scale=1.25, tokens=[0, 1, 2, V - 1])


def test_a_logit_that_becomes_infinite_is_seen(ctx):
    x = np.random.default_rng(0).standard_normal((2, 3000)).astype(np.float32)
    x[0, 2000] = 3e38
    ids, top, lp, ent = ctx.alloc_n(np.uint32, 4), ctx.alloc_n(np.float32, 4), ctx.alloc_n(np.float32, 2), ctx.alloc_n(np.float32, 2)
    ctx.token_logprobs(ctx.upload_new(x), F32, 2, 3000, scale=1.5, tokens=ctx.upload_new(np.array([1, 2], np.uint32)), logprob=lp,
                       entropy=ent, k=2, top_ids=ids, top_logprobs=top)
    lp, ent, top = ctx.download(lp, np.float32, 2), ctx.download(ent, np.float32, 2), ctx.download(top, np.float32, 4)
    assert np.isnan(lp[0]) and np.isnan(ent[0]) and np.isnan(top[:2]).all()
    assert np.isfinite(lp[1]) and np.isfinite(ent[1]) and np.isfinite(top[2:]).all()
    assert ctx.download(ids, np.uint32, 4)[0] == 2000

"""Token scores and their gradient at the borders of fp32: logits masked by the type's lowest value under large weights, and
tokens that are nearly certain."""
import numpy as np
import pytest

from tsplit_b200 import ndarray, gpu_ops as ad

HALF = 2.0 ** -24            # half a step of fp32, relative


@pytest.fixture(params=[pytest.param("cpu"), pytest.param("gpu", marks=pytest.mark.gpu)])
def ctx(request):
    return None if request.param == "cpu" else ndarray.gpu(0)


def scores(x, ids, g, top, ctx):
    """(result, gradient of the logits)"""
    v = [ad.Variable(n) for n in "xig"]
    y = ad.token_log_prob_op(v[0], v[1], top_k=top)
    out = ad.Executor([y, ad.token_log_prob_gradient_op(v[0], v[1], y, v[2])], ctx=ctx).run(
        dict(zip(v, (x, ids, g))), convert_to_numpy_ret_vals=True)
    return [np.asarray(o, np.float64) for o in out]


def definition(x, ids, g, top):
    """The same in 64 bits, from deviations from the row's maximum: nothing is lost where one token is nearly certain."""
    x, rows = x.astype(np.float64), np.arange(len(x))
    u = x - x.max(1, keepdims=True)
    best = u.argmax(1)
    e = np.exp(u)
    e[rows, best] = 0
    log_z = np.log1p(e.sum(1, keepdims=True))
    e[rows, best] = 1
    lp, p = u - log_z, e * np.exp(-log_z)
    h = -np.where(p > 0, p * np.where(p > 0, lp, 0), 0).sum(1, keepdims=True)
    cols = np.argsort(-x, axis=1, kind="stable")[:, :top]
    other = -np.expm1(lp)                                              # 1 - p
    dx = p * (g[:, 2:3] - g[:, 1:2] * np.where(p > 0, lp + h, 0))
    for j in range(top + 1):
        at, w = (ids.astype(int), g[:, 0]) if j == 0 else (cols[:, j - 1], g[:, 2 + j])
        own = dx[rows, at] + w * other[rows, at]
        dx -= w[:, None] * p
        dx[rows, at] = own
    return lp[rows, ids.astype(int)], np.take_along_axis(lp, cols, 1), cols, dx


@pytest.mark.parametrize("rows,v", [(3, 20), (4, 700), (2, 3000), (2, 20000), (160, 20000), (1200, 300)])
@pytest.mark.parametrize("weight", [-3.0, 1e4])
def test_gradients_of_logits_masked_by_the_lowest_number(rows, v, weight, ctx):
    """A token that cannot be said has probability 0 and no gradient from the entropy, however large the entropy's weight:
    weight * log p alone is beyond fp32 there."""
    r = np.random.default_rng(v)
    x = r.standard_normal((rows, v)).astype(np.float32)
    x[:, 1::3] = np.finfo(np.float32).min
    ids = np.full(rows, 4.0, np.float32)                               # a masked one: its own weight, and no more
    ids[::2] = 0
    g = r.standard_normal((rows, 3 + 2 * 2)).astype(np.float32)
    g[:, 1] = weight
    _, dx = scores(x, ids, g, 2, ctx)
    _, _, cols, want = definition(x, ids, g, 2)
    assert np.isfinite(dx).all()
    masked = x == np.finfo(np.float32).min
    masked[np.arange(rows), ids.astype(int)] = False
    assert not dx[masked].any()
    given = np.flatnonzero(ids == 4)
    assert np.array_equal(dx[given, 4], g[given, 0])
    # p is off by some 20 steps (sums of 20000 terms in fixed groups, a fast exponential), and the factors of p are at most
    # |g| + |weight| (|log p| + H) <= 4 + |weight| (20 + 10)
    assert np.abs(dx - want).max() <= 64 * HALF * (4 + abs(weight) * 30)


@pytest.mark.parametrize("v", [30, 1000, 3000, 10000, 32000, 40000])
@pytest.mark.parametrize("rows", [2, 160])
@pytest.mark.parametrize("high", [12.0, 16.0, 20.0, 25.0, 90.0])
@pytest.mark.parametrize("at", [0.0, 1000.0])
def test_tokens_that_are_nearly_certain(v, rows, high, at, ctx):
    """log p of a token with p near 1 is off by a few steps of 1, not by steps of its logit, and so is 1 - p in its gradient:
    the row of the gradient adds up to nothing."""
    x = np.full((rows, v), at, np.float32)
    x[:, v // 3] = at + high
    x[:, 5] = at + 1
    ids = np.full(rows, v // 3, np.float32)
    g = np.zeros((rows, 3 + 2 * 2), np.float32)
    g[:, 0] = 1
    g[1::2, 0], g[1::2, 3] = 0, 1                                      # as the given token, and as the likeliest one
    out, dx = scores(x, ids, g, 2, ctx)
    lp, best, cols, want = definition(x, ids, g, 2)
    # Z in [1, 2): a sum of up to 32 terms of a thread (of long rows: v / 256), then some 24 joins, each off by 2^-24; fast
    # exponentials are off by 2 + 1.2 |u| steps of what the others add; log p at the maximum is -log Z, rounded once
    rest = np.expm1(-lp)[:, None]
    step = HALF * (64 + v / 256 + (8 + 3 * high) * rest)
    assert np.all(np.abs(out[:, 0] - lp) <= step[:, 0] + 2 * HALF * np.abs(lp))
    assert np.all(np.abs(out[:, 3] - best[:, 0]) <= step[:, 0] + 2 * HALF * np.abs(best[:, 0]))
    assert np.all(np.abs(out[:, 4] - best[:, 1]) <= step[:, 0] + 8 * HALF * np.abs(best[:, 1]))
    own = dx[np.arange(rows), v // 3]
    assert np.all(np.abs(own - want[np.arange(rows), v // 3]) <= step[:, 0] + 8 * HALF * np.abs(own))
    # the others: p from logit - log-sum-exp, which is off by half a step of the largest
    rel = HALF * (80 + 4 * (abs(at) + high) + v / 256)
    others = np.delete(np.arange(v), v // 3)
    assert np.all(np.abs(dx[:, others] - want[:, others]) <= rel * np.abs(want[:, others]) + 1e-37)

"""Scaled embedding lookup with its gradient by sorted tokens, and log probabilities of given tokens: the NumPy path and
the kernels against plain formulas in 64 bits, at the sizes and values where they can go wrong."""
import numpy as np
import pytest

from tsplit_b200 import ndarray, gpu_ops as ad

HALF = 2.0 ** -24            # half a step of fp32, relative


@pytest.fixture(params=[pytest.param("cpu"), pytest.param("gpu", marks=pytest.mark.gpu)])
def ctx(request):
    return None if request.param == "cpu" else ndarray.gpu(0)


def rng(*key):
    return np.random.default_rng([abs(int(k)) for k in key])


def evaluate(build, feeds, ctx, **kw):
    names, nodes = build()
    ex = ad.Executor(nodes, ctx=ctx, **kw)
    out = ex.run({names[k]: v for k, v in feeds.items()}, convert_to_numpy_ret_vals=True)
    return [np.asarray(o).astype(np.float64) for o in out]


# ------------------------------------------------------------------------------------------------ embedding
def embed_graph(scale, padding):
    def build():
        t, i, g = ad.Variable("table"), ad.Variable("ids"), ad.Variable("g")
        y = ad.scaled_embedding_op(t, i, scale=scale, padding_id=padding)
        return {"table": t, "ids": i, "g": g}, [y, ad.scaled_embedding_gradient_op(g, i, t, scale=scale, padding_id=padding)]
    return build


def check_embed(table, ids, g, scale, padding, ctx, **kw):
    y, dt = evaluate(embed_graph(scale, padding), {"table": table, "ids": ids, "g": g}, ctx, **kw)
    v, d = table.shape
    flat, rows = ids.reshape(-1).astype(np.int64), g.reshape(-1, d).astype(np.float64)
    known = (flat >= 0) & (flat < v)
    want = np.where(known[:, None], table.astype(np.float64)[np.where(known, flat, 0)] * np.float32(scale), 0)
    assert np.all(np.abs(y.reshape(-1, d) - want) <= HALF * np.abs(want))
    known &= flat != (padding if padding is not None else -1)
    want, size, count = np.zeros((v, d)), np.zeros((v, d)), np.zeros(v)
    np.add.at(want, flat[known], rows[known])
    np.add.at(size, flat[known], np.abs(rows[known]))
    np.add.at(count, flat[known], 1)
    # each of the count - 1 additions and the product round once
    assert np.all(np.abs(dt - want * np.float32(scale)) <= (count[:, None] + 1) * HALF * size * abs(np.float32(scale)) * 1.001)
    return y, dt


@pytest.mark.parametrize("n,v,d", [(1, 1, 1), (1, 5, 4), (7, 3, 8), (37, 500, 128), (16, 40, 4), (17, 40, 5), (300, 257, 33), (4096, 300, 8),
                                   (4097, 255, 4), (5000, 65536, 4), (9001, 100, 129)])
@pytest.mark.parametrize("padding", [None, 0])
def test_embedding_and_its_gradient(n, v, d, padding, ctx):
    r = rng(n, v, d)
    ids = r.integers(0, v, n).astype(np.float32)
    check_embed(r.standard_normal((v, d), np.float32), ids, r.standard_normal((n, d), np.float32), 2.5, padding, ctx)


@pytest.mark.gpu
@pytest.mark.parametrize("n,v,d", [(8192, 32000, 64), (16384, 1000, 12), (16385, 1000, 12), (32768, 70000, 4), (32769, 70000, 4), (40000, 256, 7),
                                   (70000, 255, 16), (100001, 1 << 20, 4), (131072, 64000, 36)])
def test_embedding_of_many_tokens(n, v, d):
    r = rng(n, v, d)
    ids = np.exp(r.random(n) * np.log(v)).astype(np.int64).astype(np.float32)
    ids[r.random(n) < 0.2] = 0
    check_embed(r.standard_normal((v, d), np.float32), ids, r.standard_normal((n, d), np.float32), 0.5, None, ndarray.gpu(0))


@pytest.mark.gpu
@pytest.mark.parametrize("n,v,d", [(37887, 90, 33), (37889, 90, 33), (37888, 90, 128), (37890, 50, 127), (37891, 50, 132), (70, 90, 31), (70, 90, 1023),
                                   (9, 70, 4100)])
def test_lookups_of_whole_rows(n, v, d):
    """Rows of fewer and of more than 32 pieces, one and several to a warp, ids outside among them."""
    r = rng(n, v, d)
    ids = r.integers(-2, v + 2, n).astype(np.float32)
    check_embed(r.standard_normal((v, d), np.float32), ids, r.standard_normal((n, d), np.float32), 3.0, 1, ndarray.gpu(0))


@pytest.mark.parametrize("what", ["same", "none", "padding", "outside", "falling", "runs"])
@pytest.mark.parametrize("n", [33, 1500, pytest.param(40000, marks=pytest.mark.gpu)])
def test_embedding_of_unusual_ids(what, n, ctx):
    v, d = 97, 12
    r = rng(n, len(what))
    ids = {"same": np.full(n, 5), "none": np.full(n, -1), "padding": np.where(np.arange(n) % 3 == 0, 7, 96), "outside":
           r.integers(-50, 200, n), "falling": 96 - np.arange(n) * 97 // n, "runs": np.repeat(r.integers(0, v, n // 11 + 1), 11)[:n]}[what]
    check_embed(r.standard_normal((v, d), np.float32), ids.astype(np.float32), r.standard_normal((n, d), np.float32), 1.0, 7, ctx)


@pytest.mark.parametrize("n,v,d", [(1, 64000, 8), (2, 3, 130), (511, 100, 5), (512, 1, 33), (512, 2000, 132), (513, 2000, 132),
                                   (300, 70001, 12), (400, 40, 260), (500, 1100000, 4)])
@pytest.mark.parametrize("what", ["spread", "skewed", "two"])
def test_embedding_gradient_of_a_few_tokens(n, v, d, what, ctx):
    """Around the length up to which tokens are not sorted; rows that few, more than 32 or all positions have."""
    r = rng(n, v, d)
    ids = {"spread": r.integers(0, v, n), "skewed": np.exp(r.random(n) * np.log(v)).astype(np.int64),
           "two": np.where(r.random(n) < 0.9, v - 1, 0)}[what]
    check_embed(r.standard_normal((v, d), np.float32), ids.astype(np.float32), r.standard_normal((n, d), np.float32), -1.5, None, ctx)


def test_embedding_of_no_number_is_outside(ctx):
    ids = np.array([np.nan, np.inf, -np.inf, 1e30, 2], np.float32)
    if ctx is None:
        ids[:4] = -1                     # (NumPy's conversion of those is undefined)
    y, dt = evaluate(embed_graph(1.0, None), {"table": np.ones((3, 4), np.float32), "ids": ids, "g": np.ones((5, 4), np.float32)}, ctx)
    assert np.array_equal(y, np.array([[0], [0], [0], [0], [1]]) * np.ones((1, 4)))
    assert np.array_equal(dt, np.array([[0], [0], [1]]) * np.ones((1, 4)))


def test_embedding_keeps_the_shape_of_its_ids_and_its_gradient_in_a_graph(ctx):
    r = rng(3)
    table, ids = r.standard_normal((11, 6), np.float32), r.integers(0, 11, (2, 5)).astype(np.float32)
    w = r.standard_normal((2, 5, 6), np.float32)

    def build():
        t, i, k = ad.Variable("t"), ad.Variable("i"), ad.Variable("w")
        y = ad.scaled_embedding_op(t, i, scale=3.0, padding_id=4)
        return {"t": t, "i": i, "w": k}, [y] + ad.gradients(ad.reduce_sum_op(ad.mul_op(y, k), [0, 1, 2]), [t])
    y, dt = evaluate(build, {"t": table, "i": ids, "w": w}, ctx)
    assert y.shape == (2, 5, 6)
    want = np.zeros((11, 6))
    np.add.at(want, ids.astype(int)[ids != 4], 3.0 * w[ids != 4].astype(np.float64))
    assert np.allclose(dt, want, rtol=0, atol=12 * HALF * 3 * np.abs(w).max())


def test_embedding_refuses(ctx):
    def build(ts, gs):
        t, i, g = ad.Variable("t"), ad.Variable("i"), ad.Variable("g")
        feeds = {"t": np.ones(ts, np.float32), "i": np.zeros((2, 3), np.float32), "g": np.ones(gs, np.float32)}
        return lambda: ({"t": t, "i": i, "g": g}, [ad.scaled_embedding_op(t, i), ad.scaled_embedding_gradient_op(g, i, t)]), feeds
    for ts, gs in [((4, 5, 6), (2, 3, 6)), ((4, 5), (2, 3, 4)), ((4, 5), (6, 5))]:
        with pytest.raises(AssertionError):
            evaluate(*build(ts, gs), ctx)


def test_embedding_refuses_what_is_not_row_major():
    import torch
    from tsplit_b200.ops import _gpu as G
    a = ndarray.NDArray(torch.zeros(6, 8)[:, ::2], ndarray.cpu(0))
    ok = ndarray.empty((6, 4))
    for args in [(a, ndarray.empty((6,)), ok), (ok, ndarray.empty((6,)), a)]:
        with pytest.raises(ValueError, match="row-major"):
            G.scaled_embedding(*args, 1.0, None)
        with pytest.raises(ValueError, match="row-major"):
            G.scaled_embedding_grad(*args, 1.0, None, None)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [5000, 50000])
def test_embedding_gradient_has_the_same_bits_every_time_and_on_unaligned_rows(n):
    import torch
    from tsplit_b200.ops import _gpu as G
    from tsplit_b200.stream import create_stream_handle
    ctx = ndarray.gpu(0)
    st = create_stream_handle(ctx)
    arr = lambda t: ndarray.from_tensor(t, ctx)
    g = torch.randn(n * 16 + 1, device="cuda")
    ids = torch.randint(0, 50, (n,), device="cuda").float()
    rows = g[:-1].view(n, 16)
    out = [torch.empty(50, 16, device="cuda") for _ in range(4)]
    shifted = torch.empty(n * 16 + 1, device="cuda")[1:].view(n, 16).copy_(rows)
    torch.cuda.synchronize()
    for o in out[:3]:
        G.scaled_embedding_grad(arr(rows), arr(ids), arr(o), 1.5, None, st)
    G.scaled_embedding_grad(arr(shifted), arr(ids), arr(out[3]), 1.5, None, st)        # the same sums, 4 bytes at a time
    st.sync()
    for o in out[1:]:
        assert torch.equal(out[0], o)


@pytest.mark.gpu
def test_embedding_gradients_of_two_captured_steps_that_alternate():
    """Two executors with streams and scratch of their own, replayed in turn with new values; a bigger one in between."""
    ctx = ndarray.gpu(0)
    r = rng(8)
    steps = []
    for n, v, d in [(3000, 200, 16), (700, 90, 8), (40000, 300, 8)]:
        names, nodes = embed_graph(1.0, 0)()
        steps.append((n, v, d, names, ad.Executor(nodes, ctx=ctx, use_graph=True)))
    for _ in range(4):
        for n, v, d, names, ex in steps:
            ids, g = r.integers(0, v, n).astype(np.float32), r.standard_normal((n, d), np.float32)
            _, dt = ex.run({names["table"]: np.zeros((v, d), np.float32), names["ids"]: ids, names["g"]: g}, convert_to_numpy_ret_vals=True)
            want, size = np.zeros((v, d)), np.zeros((v, d))
            np.add.at(want, ids.astype(int), g * (ids != 0)[:, None])
            np.add.at(size, ids.astype(int), np.abs(g))
            assert np.all(np.abs(dt - want) <= (n * v ** -0.5 + 20) * HALF * size + 1e-30)


# ------------------------------------------------------------------------------------------------ log probabilities
def score_exact(x, ids, top):
    """(out, p, log p) by the definition, in 64 bits."""
    x = x.astype(np.float64)
    m = x.max(1, keepdims=True)
    lse = (m + np.log(np.exp(x - m).sum(1, keepdims=True)))
    logs = x - lse
    p = np.exp(logs)
    h = -np.where(p > 0, p * np.where(p > 0, logs, 0), 0).sum(1)
    out = np.zeros((len(x), 3 + 2 * top))
    given = (ids >= 0) & (ids < x.shape[1])
    out[given, 0] = logs[np.flatnonzero(given), ids[given].astype(int)]
    out[:, 1], out[:, 2] = h, lse[:, 0]
    for r in range(len(x)):
        best = sorted(range(x.shape[1]), key=lambda c: (-x[r, c], c))[:top]
        out[r, 3:3 + top], out[r, 3 + top:] = logs[r, best], best
    return out, p, logs


def score_graph(top):
    def build():
        x, i, g = ad.Variable("x"), ad.Variable("i"), ad.Variable("g")
        y = ad.token_log_prob_op(x, i, top_k=top)
        return {"x": x, "i": i, "g": g}, [y, ad.token_log_prob_gradient_op(x, i, y, g)]
    return build


def check_score(x, ids, top, g, ctx, **kw):
    out, dx = evaluate(score_graph(top), {"x": x, "i": ids, "g": g}, ctx, **kw)
    want, p, logs = score_exact(x, ids, top)
    v, g = x.shape[1], g.astype(np.float64)
    big = np.abs(np.where(np.isfinite(x), x, 0)).max()
    # a fast exponential is off by 2 + 1.2 |u| steps, weighted by p; a thread adds max(32, v / 256) terms and some 20 joins
    # follow; x - max, the log-sum-exp and log p round once each
    tol = 2 * HALF * (4 + 2 * np.log(v + 1) + (max(32, v / 256) + 24) / 2 + 3 * big)
    wide = tol * (2 + np.log(v + 1))
    for cols, t in [(slice(0, 1), tol), (slice(1, 2), wide), (slice(2, 3 + top), tol)]:
        a, b = out[:, cols], want[:, cols]
        assert np.array_equal(np.isinf(a), np.isinf(b)) and np.all(np.abs(np.where(np.isinf(b), 0, a - np.where(np.isinf(b), 0, b)))[np.isfinite(b)] <= t)
    assert np.array_equal(out[:, 3 + top:], want[:, 3 + top:])
    given = (ids >= 0) & (ids < v)
    w = np.zeros_like(x, dtype=np.float64)
    rows = np.arange(len(x))
    w[rows[given], ids[given].astype(int)] += g[given, 0]
    for j in range(top):
        w[rows, want[:, 3 + top + j].astype(int)] += g[:, 3 + j]
    total, lp = w.sum(1, keepdims=True), np.where(p > 0, logs, 0)
    dwant = w - p * total + g[:, 2:3] * p - g[:, 1:2] * p * (lp + want[:, 1:2])
    size = np.abs(w) + p * (np.abs(w).sum(1, keepdims=True) + np.abs(g[:, 2:3]) + np.abs(g[:, 1:2]) * (np.abs(lp) + want[:, 1:2] + 1))
    # p is off by the log probability's error and its exponential's steps; the rest are a few roundings of each term
    assert np.all(np.abs(dx - dwant) <= size * (2 * wide + 2 * HALF * (8 + 3 * np.abs(lp))) + 1e-37)
    return out, dx


def score_case(rows, v, top, seed=0, spread=3.0, masked=True):
    r = rng(rows, v, top, seed)
    x = (r.standard_normal((rows, v)) * spread).astype(np.float32)
    if masked and v > 40:
        x[:, 3::7] = -np.inf
    ids = r.integers(0, v, rows).astype(np.float32)
    ids[rows // 2] = -1
    ids[rows // 3] = v
    return x, ids, r.standard_normal((rows, 3 + 2 * top)).astype(np.float32)


@pytest.mark.parametrize("rows,v", [(1, 1), (1, 7), (3, 2), (5, 33), (4, 257), (7, 1000), (2, 1023), (3, 4097), (1, 10007)])
@pytest.mark.parametrize("top", [0, 1, 5, 32])
def test_scores_of_tokens(rows, v, top, ctx):
    x, ids, g = score_case(rows, v, min(top, v))
    check_score(x, ids, min(top, v), g, ctx)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,v,top", [(1, 128001, 20), (2, 32000, 32), (9, 32000, 7), (80, 5000, 3), (300, 2047, 32), (2000, 31, 8),
                                        (75, 8191, 16)])
def test_scores_of_long_and_of_many_rows(rows, v, top):
    x, ids, g = score_case(rows, v, top)
    check_score(x, ids, top, g, ndarray.gpu(0))


@pytest.mark.parametrize("v", [64, 700, 9000])
@pytest.mark.parametrize("kind", ["rising", "falling", "equal", "two", "peak", "zeros", "last"])
def test_alternatives_of_unusual_rows(kind, v, ctx):
    """Orders that make every column a candidate, ties, and a row where one token is nearly certain."""
    c = np.arange(v)
    x = {"rising": c * 2.0 ** -9, "falling": -c * 2.0 ** -9, "equal": np.full(v, 1.25), "two": np.where(c % 5 == 2, 3.0, 1.0),
         "peak": np.where(c == v // 2, 40.0, 0.0), "zeros": np.where(c % 2 == 0, -0.0, 0.0), "last": np.where(c >= v - 3, 7.0, -2.0)}[kind]
    x = np.stack([x, x[::-1]]).astype(np.float32)
    ids = np.array([v // 2, 0], np.float32)
    g = rng(v).standard_normal((2, 3 + 2 * 11)).astype(np.float32)
    check_score(x, ids, 11, g, ctx)


@pytest.mark.gpu
@pytest.mark.parametrize("v", [31, 32, 33, 128, 129, 512, 513, 1024, 1025, 2048, 2049, 4096, 4097, 6144, 6145, 8192, 8193, 12288, 12289, 16384,
                               16385, 32768, 32769])
@pytest.mark.parametrize("rows,top", [(3, 0), (5, 17), (150, 1), (150, 32)])
def test_scores_at_the_borders_between_layouts(rows, v, top):
    """Rows of one warp, of several, of a block, of a cluster, and the number of rows from which another is taken."""
    top = min(top, v)
    x, ids, g = score_case(rows, v, top)
    check_score(x, ids, top, g, ndarray.gpu(0))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,v,top", [(1183, 40, 5), (1184, 40, 5), (1185, 2047, 3), (1184, 2048, 32), (1190, 2049, 1), (3001, 700, 0)])
def test_gradients_of_many_short_rows(rows, v, top):
    x, ids, g = score_case(rows, v, top)
    check_score(x, ids, top, g, ndarray.gpu(0))


@pytest.mark.gpu
@pytest.mark.parametrize("v", [30, 1000, 2000, 5000, 20000])
@pytest.mark.parametrize("top", [1, 32])
def test_alternatives_of_many_equal_and_missing_logits(v, top):
    """More columns that reach the bound than there is room for, and rows with fewer numbers than alternatives."""
    top = min(top, v)
    x = np.full((6, v), 2.5, np.float32)
    x[1, : v // 2] = -np.inf
    x[2] = -np.inf
    x[3] = np.nan
    x[4, 1:] = np.nan
    x[5, ::3] = 9.0
    ids = np.array([0, v - 1, 3, 4, 0, v + 5], np.float32)
    feeds = {"x": x, "i": ids, "g": np.ones((6, 3 + 2 * top), np.float32)}
    want = evaluate(score_graph(top), feeds, None)[0]
    got = evaluate(score_graph(top), feeds, ndarray.gpu(0))[0]
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[:, 3 + top:], want[:, 3 + top:])
    assert np.allclose(got, want, rtol=0, atol=1e-5, equal_nan=True)          # (numbers of size 10: 10 steps of 2^-20 each)


def test_rows_of_masked_logits(ctx):
    """Rows with fewer tokens that can be said than alternatives are asked for, and none at all."""
    x = np.full((4, 300), -np.inf, np.float32)
    x[0, [7, 200]] = [1.0, 2.0]
    x[1, 299] = -3.0
    x[2, ::2] = np.finfo(np.float32).min
    ids = np.array([7, 0, 4, 9], np.float32)
    g = rng(5).standard_normal((4, 3 + 8)).astype(np.float32)
    out, dx = evaluate(score_graph(4), {"x": x, "i": ids, "g": g}, ctx)
    assert np.array_equal(out[:, 7:], [[200, 7, 0, 1], [299, 0, 1, 2], [0, 2, 4, 6], [0, 1, 2, 3]])
    assert np.isneginf(out[0, 5:7]).all() and out[1, 0] == -np.inf and out[1, 1] == 0 and out[1, 2] == -3 and out[1, 3] == 0
    assert out[3, 0] == out[3, 2] == -np.inf and out[3, 1] == 0 and np.isneginf(out[3, 3:7]).all() and not dx[3].any()
    assert np.allclose(out[2, 1], np.log(150), rtol=0, atol=200 * HALF) and np.isfinite(dx[2]).all()
    lse = np.log(np.exp(1.0) + np.exp(2.0))
    assert np.allclose(out[0, [0, 2, 3, 4]], [1 - lse, lse, 2 - lse, 1 - lse], rtol=0, atol=40 * HALF)
    assert np.isfinite(dx[:3]).all() and dx[1, 0] == g[1, 0] + g[1, 4]          # a masked column has its own weights only


def test_no_number_among_the_logits(ctx):
    x = np.zeros((3, 50), np.float32)
    x[0, 4] = np.nan
    x[1, :] = np.nan
    x[1, 9] = 2.0
    x[2, 3] = np.inf
    out, dx = evaluate(score_graph(3), {"x": x, "i": np.zeros(3, np.float32), "g": np.ones((3, 9), np.float32)}, ctx)
    assert np.isnan(out[:, :6]).all() and np.isnan(dx).all(1).tolist() == [True] * 3
    assert np.array_equal(out[:, 6:], [[0, 1, 2], [9, -1, -1], [3, 0, 1]])


@pytest.mark.parametrize("top", [0, 3])
def test_gradient_of_scores_by_differences(top):
    """The NumPy gradient against central differences of the definition in 64 bits."""
    x, ids, g = score_case(4, 23, top, masked=False)
    _, dx = evaluate(score_graph(top), {"x": x, "i": ids, "g": g}, None)
    g = g.astype(np.float64)
    g[:, 3 + top:] = 0
    h = 1e-4
    for r in range(4):
        for c in range(23):
            up, down = x.astype(np.float64), x.astype(np.float64)
            up[r, c] += h
            down[r, c] -= h
            d = ((score_exact(up, ids, top)[0] - score_exact(down, ids, top)[0]) * g).sum() / (2 * h)
            assert abs(d - dx[r, c]) <= 1e-5         # h^2 / 6 times a third derivative of a few units; rounding 2^-53 * 20 / h


def test_scores_in_a_training_graph(ctx):
    """Slices of the result, a loss of them, and the gradient of the product that made the logits."""
    r = rng(4)
    h, w, ids = r.standard_normal((12, 16), np.float32), r.standard_normal((16, 40), np.float32), r.integers(0, 40, 12).astype(np.float32)

    def build():
        a, b, i = ad.Variable("h"), ad.Variable("w"), ad.Variable("i")
        y = ad.token_log_prob_op(ad.matmul_op(a, b), ad.array_reshape_op(i, (3, 4)), top_k=2)
        logp, entropy = ad.slice_op(y, (0, 0), (12, 1)), ad.slice_op(y, (0, 1), (12, 1))
        loss = ad.reduce_sum_op(ad.addbyconst_op(ad.opposite_op(logp), 0.0) + ad.mul_byconst_op(entropy, -0.1), [0, 1])
        return {"h": a, "w": b, "i": i}, [loss] + ad.gradients(loss, [b])
    loss, dw = evaluate(build, {"h": h, "w": w, "i": ids}, ctx)
    x = h.astype(np.float64) @ w
    want, p, logs = score_exact(x, ids, 0)
    dx = p + 0.1 * p * (logs + want[:, 1:2])
    dx[np.arange(12), ids.astype(int)] -= 1
    # the product on the GPU takes ten bits of each factor: 2^-11 a factor, over 16 terms of up to some units
    assert np.allclose(loss, (-want[:, 0] - 0.1 * want[:, 1]).sum(), rtol=0, atol=12 * 0.05)
    assert np.allclose(dw, h.T.astype(np.float64) @ dx, rtol=0, atol=0.05)


def test_scores_refuse(ctx):
    with pytest.raises(AssertionError):
        ad.token_log_prob_op(ad.Variable("x"), ad.Variable("i"), top_k=33)
    with pytest.raises(AssertionError):
        ad.token_log_prob_op(ad.Variable("x"), ad.Variable("i"), top_k=-1)
    for xs, n, top, gs in [((4, 5, 6), 20, 0, (4, 3)), ((4, 5), 3, 0, (4, 3)), ((4, 5), 4, 6, (4, 15)), ((4, 5), 4, 1, (4, 3))]:
        with pytest.raises(AssertionError):
            evaluate(score_graph(top), {"x": np.zeros(xs, np.float32), "i": np.zeros(n, np.float32), "g": np.zeros(gs, np.float32)}, ctx)


def test_scores_refuse_what_is_not_row_major():
    import torch
    from tsplit_b200.ops import _gpu as G
    x = ndarray.NDArray(torch.zeros(8, 6).t(), ndarray.cpu(0))
    ids, out, ok = ndarray.empty((6,)), ndarray.empty((6, 3)), ndarray.empty((6, 8))
    with pytest.raises(ValueError, match="row-major"):
        G.token_score(x, ids, out, 0, None)
    with pytest.raises(ValueError, match="row-major"):
        G.token_score_grad(ok, ids, out, out, x, None)


@pytest.mark.gpu
def test_scores_of_rows_that_begin_anywhere():
    """Rows at every offset from a 16-byte boundary, in and out apart."""
    import torch
    from tsplit_b200.ops import _gpu as G
    from tsplit_b200.stream import create_stream_handle
    ctx = ndarray.gpu(0)
    st = create_stream_handle(ctx)
    arr = lambda t: ndarray.from_tensor(t, ctx)
    x, ids, g = score_case(5, 1003, 4)
    want = None
    for a in range(4):
        for b in range(4):
            xt = torch.empty(5 * 1003 + 8, device="cuda")[a:a + 5 * 1003].view(5, 1003).copy_(torch.from_numpy(x))
            dx = torch.empty(5 * 1003 + 8, device="cuda")[b:b + 5 * 1003].view(5, 1003)
            out, i, gt = torch.empty(5, 11, device="cuda"), torch.from_numpy(ids).cuda(), torch.from_numpy(g).cuda()
            torch.cuda.synchronize()
            G.token_score(arr(xt), arr(i), arr(out), 4, st)
            G.token_score_grad(arr(xt), arr(i), arr(out), arr(gt), arr(dx), st)
            st.sync()
            got = torch.cat([out, dx], 1).cpu().numpy()
            if want is None:
                want, p, logs = score_exact(x, ids, 4)
                first = got
            assert np.allclose(got[:, :7][np.isfinite(want[:, :7])], want[:, :7][np.isfinite(want[:, :7])], rtol=0, atol=1e-5)
            assert np.allclose(got[:, 11:], first[:, 11:], rtol=0, atol=1e-5)

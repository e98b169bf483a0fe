"""The operators around the attention stack used together: in the Transformer, trained and scored, under every kind of
executor, and in a decoder that takes one token at a time."""
import numpy as np
import pytest

from tsplit_b200 import ndarray, gpu_ops as ad, optimizer
from tsplit_b200.models import transformer

SIZES = dict(vocab_size=60, d_model=32, num_heads=4, d_ff=48, num_blocks=1, maxlen1=9, maxlen2=8, batch_size=4)


@pytest.fixture(params=[pytest.param("cpu"), pytest.param("gpu", marks=pytest.mark.gpu)])
def ctx(request):
    return None if request.param == "cpu" else ndarray.gpu(0)


def model(**kw):
    return transformer(**{**SIZES, "scaled_embedding": True, "cross_attention": True, "seed": 11, **kw})


def batch(m, padded=True):
    f = m.synthetic_batch(4)
    if padded:                       # sentences of their own lengths; the last one is padding all through
        for b in range(m.hp.batch_size):
            f[m.xs][b, m.hp.maxlen1 - 2 * b:] = 0
            f[m.ys_in][b, m.hp.maxlen2 - 1 - b:] = 0
        f[m.xs][m.hp.batch_size - 1] = 0
    return f


def evaluate(nodes, feed, ctx, cls=None, steps=1, **kw):
    ex = (cls or ad.Executor)(nodes, ctx=ctx, **kw)
    for _ in range(steps):
        out = ex.run(feed, convert_to_numpy_ret_vals=True)
    return [np.asarray(o, dtype=np.float64) if o is not None else None for o in out]


def same_step(got, want, ctx, what):
    """Loss (first) and gradients of a whole network.  On the GPU its products keep 2^-11 of each factor, so a pre-activation
    nearer to zero than that share of its terms may fall on the other side of the ReLU, which takes a whole term of a gradient in
    or out: no bound holds element by element.  Loss and direction have to agree, as for the other networks' steps."""
    if ctx is None:
        for n, g, w in zip(what, got, want):
            assert np.abs(g - w).max() <= 3e-5 * np.abs(w).max(), n
        return
    assert np.abs(got[0] - want[0]).max() <= 5e-2 * np.abs(want[0]).max()
    a, b = (np.concatenate([g.reshape(-1) for g in v[1:]]) for v in (got, want))
    assert np.isfinite(a).all() and a @ b > 0.98 * np.linalg.norm(a) * np.linalg.norm(b)


def test_the_model_is_the_one_of_separate_operators(ctx):
    """With the key and value projections side by side in one, loss and gradients are those of the model without options."""
    plain = transformer(**SIZES, seed=11)
    ours = model()
    by_name = {v.name: v for v in plain.variables}
    for v in ours.variables:
        n = v.name.replace("_kv_", "_k_")
        value = by_name[n].tensor_value
        if "_kv_" in v.name:
            value = np.concatenate([value, by_name[n.replace("_k_", "_v_")].tensor_value], axis=-1)
        v.tensor_value = np.ascontiguousarray(value)
    names = [v.name for v in plain.variables if not v.name.endswith("_k_bias")]
    a = evaluate([plain.loss] + ad.gradients(plain.loss, [by_name[n] for n in names]), batch(plain, False), None)
    mine = {v.name: v for v in ours.variables}
    b = evaluate([ours.loss] + ad.gradients(ours.loss, list(mine.values())), batch(ours, False), ctx)
    got = dict(zip(["loss"] + list(mine), b))
    for n in [n for n in got if "_kv_" in n]:
        k, v = np.split(got.pop(n), 2, axis=-1)
        got[n.replace("_kv_", "_k_")], got[n.replace("_kv_", "_v_")] = k, v
    names = ["loss"] + names
    same_step([got[n] for n in names], a, ctx, names)


def scored(m, top=3):
    """A loss of token scores: likelihood with a bonus for entropy, a penalty on the log-sum-exp and one on the best alternative."""
    s = m.token_scores(top)
    rows = m.hp.batch_size * (m.hp.maxlen2 - 1)
    parts = [ad.mul_byconst_op(ad.slice_op(s, (0, c), (rows, 1)), w) for c, w in ((0, -1.0), (1, -0.05), (2, 0.01), (3, 0.02))]
    total = parts[0]
    for p in parts[1:]:
        total = total + p
    return s, ad.mul_byconst_op(ad.reduce_sum_op(total, [0, 1]), 1.0 / rows)


def test_a_step_that_trains_on_scores(ctx):
    """Tokens in, attention across, tokens out, and every gradient: against the NumPy path."""
    def build():
        m = model()
        s, loss = scored(m)
        return [loss, s] + ad.gradients(loss, m.variables), batch(m)
    want, got = evaluate(*build(), None), evaluate(*build(), ctx)
    assert got[1].shape == want[1].shape and np.isfinite(got[1]).all()
    if ctx is None:
        assert np.array_equal(got[1], want[1])
    same_step([got[0]] + got[2:], [want[0]] + want[2:], ctx, range(len(got) - 1))


@pytest.mark.parametrize("graph", [False, pytest.param(True, marks=pytest.mark.gpu)])
@pytest.mark.parametrize("kind", ["base", "stream", "recompute", "vdnn", "superneurons", "capuchin", "tsplit"])
def test_every_executor_takes_the_step(kind, graph, ctx):
    """Two steps of momentum under each memory policy end where the NumPy path ends."""
    if graph and (ctx is None or kind not in ("base", "recompute", "tsplit")):
        pytest.skip("this executor does not replay")
    cls = {"base": ad.Executor, "stream": ad.StreamExecutor, "recompute": ad.recomputeExecutor, "vdnn": ad.vdnnExecutor,
           "superneurons": ad.superNeuronsExecutor, "capuchin": ad.capuchinExecutor, "tsplit": ad.microopExecutor}[kind]

    def run(cls, ctx, **kw):
        m = model(maxlen1=6)
        opt = optimizer.MomentumOptimizer(0.05, 0.9, ctx=ctx)
        _, loss = scored(m)
        train = opt.minimize(loss)
        ex = cls([loss, train], ctx=ctx, **kw)
        f = batch(m)
        losses = [float(np.asarray(ex.run(f, convert_to_numpy_ret_vals=True)[0]).reshape(-1)[0]) for _ in range(4)]
        return losses, [np.asarray(p.asnumpy() if isinstance(p, ndarray.NDArray) else p, np.float64) for p in opt.params]
    if ctx is None:
        ctx = ndarray.simgpu(0)
    kw = {"use_graph": True} if graph else {}
    (l1, p1), (l2, p2) = run(ad.Executor, None), run(cls, ctx, **kw)
    tol = 1e-5 if ctx.device_type == 3 else 0.02
    assert np.allclose(l1, l2, rtol=0, atol=tol * np.abs(l1).max())
    for a, b in zip(p1, p2):
        assert np.abs(a - b).max() <= tol * max(1.0, np.abs(a).max())


def test_two_sizes_of_one_graph_in_turn(ctx):
    """The same nodes at two feed shapes, each with an executor of its own, one after the other and again."""
    q, kv, key, g = (ad.Variable(v) for v in ("q", "kv", "key", "g"))
    y = ad.cross_attention_op(q, kv, key)
    nodes = [y] + ad.cross_attention_gradient_op(y, g)
    graph = {"use_graph": True} if ctx is not None else {}
    ex = [ad.Executor(nodes, ctx=ctx, **graph) for _ in range(2)]
    r = np.random.default_rng(5)
    feeds = [{q: r.standard_normal((2, t, 2, 16), np.float32), kv: r.standard_normal((2, 30, 2, 2, 16), np.float32),
              key: np.ones((2, 30), np.float32), g: r.standard_normal((2, t, 2, 16), np.float32)} for t in (40, 12)]
    want = [evaluate(nodes, f, None) for f in feeds]
    for _ in range(4):
        for e, f, w in zip(ex, feeds, want):
            for a, b in zip(e.run(f, convert_to_numpy_ret_vals=True), w):
                assert np.abs(a - b).max() <= 1e-5 * np.abs(b).max()


@pytest.mark.parametrize("shared", [4, 1])
def test_one_token_at_a_time_gives_what_the_whole_sentence_gives(shared, ctx):
    """A decoder that keeps the encoder's projected states and asks for one position (and for three) at a time."""
    r = np.random.default_rng(9)
    n, tq, tk, h, d = 3, 12, 50, 4, 16
    table, wq, wo = (r.standard_normal(s, np.float32) * 0.3 for s in ((40, h * d), (h * d, h * d), (h * d, 40)))
    states, ids, key = r.standard_normal((n, tk, 2, shared, d), np.float32), r.integers(0, 40, (n, tq)).astype(np.float32), np.ones((n, tk), np.float32)
    key[1, 30:] = 0
    key[2] = 0

    def build(length):
        t, i, s, k, a, b = (ad.Variable(v) for v in ("t", "i", "s", "k", "a", "b"))
        x = ad.matmul_op(ad.array_reshape_op(ad.scaled_embedding_op(t, i, scale=2.0), (n * length, h * d)), a)
        y = ad.cross_attention_op(ad.array_reshape_op(x, (n, length, h, d)), s, k)
        return ad.token_log_prob_op(ad.matmul_op(ad.array_reshape_op(y, (n * length, h * d)), b), i, top_k=2), (t, i, s, k, a, b)
    out, v = build(tq)
    whole = evaluate([out], dict(zip(v, (table, ids, states, key, wq, wo))), ctx)[0].reshape(n, tq, -1)
    for step in (1, 3):
        out, v = build(step)
        ex = ad.Executor([out], ctx=ctx, **({"use_graph": True} if ctx is not None else {}))
        for t in range(0, tq, step):
            got = ex.run(dict(zip(v, (table, np.ascontiguousarray(ids[:, t:t + step]), states, key, wq, wo))), convert_to_numpy_ret_vals=True)[0]
            # fp32 attention in both; the products around it take ten bits of each factor, in other tiles
            assert np.abs(got.reshape(n, step, -1)[..., :5] - whole[:, t:t + step, :5]).max() <= (1e-5 if ctx is None else 2e-2)

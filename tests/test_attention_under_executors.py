"""Attention across under every kind of executor: its own gradients, and what each parameter of the Transformer moves by, against
the keep-all executor's, small gradients with the same weight as large ones."""
import numpy as np
import pytest

from tsplit_b200 import ndarray, gpu_ops as ad, optimizer
from tsplit_b200.models import transformer

KINDS = {"stream": ad.StreamExecutor, "recompute": ad.recomputeExecutor, "vdnn": ad.vdnnExecutor, "superneurons": ad.superNeuronsExecutor,
         "capuchin": ad.capuchinExecutor, "tsplit": ad.microopExecutor}


@pytest.fixture(params=[pytest.param("sim"), pytest.param("gpu", marks=pytest.mark.gpu)])
def ctx(request):
    return ndarray.simgpu(0) if request.param == "sim" else ndarray.gpu(0)


def off(a, b):
    """Norm of the difference relative to the norm of ``b``."""
    a, b = np.asarray(a, np.float64), np.asarray(b, np.float64)
    assert a.shape == b.shape and np.isfinite(a).all() and np.linalg.norm(b) > 0
    return np.linalg.norm(a - b) / np.linalg.norm(b)


def attention_step(tq, tk, h, shared, d, n=3):
    """(feeds, [loss, gradients of q and kv, of their projections' weights])"""
    r = np.random.default_rng([tq, tk, h, d])
    key = r.integers(0, 3, (n, tk)).astype(np.float32)
    key[:, 0] = 1
    key[n - 1] = 0                                                   # a sentence that is padding all through
    f = {"x": r.standard_normal((n * tq, 32), np.float32), "e": r.standard_normal((n * tk, 32), np.float32),
         "wq": r.standard_normal((32, h * d), np.float32) * 0.2, "wkv": r.standard_normal((32, 2 * shared * d), np.float32) * 0.2,
         "wo": r.standard_normal((h * d, 24), np.float32) * 0.2, "key": key, "w": r.standard_normal((n * tq, 24), np.float32)}
    v = {k: ad.Variable(k) for k in f}
    q = ad.array_reshape_op(ad.matmul_op(v["x"], v["wq"]), (n, tq, h, d))
    kv = ad.array_reshape_op(ad.matmul_op(v["e"], v["wkv"]), (n, tk, 2, shared, d))
    y = ad.array_reshape_op(ad.cross_attention_op(q, kv, v["key"]), (n * tq, h * d))
    loss = ad.reduce_sum_op(ad.mul_op(ad.matmul_op(y, v["wo"]), v["w"]), [0, 1])
    return {v[k]: a for k, a in f.items()}, [loss] + ad.gradients(loss, [q, kv, v["wq"], v["wkv"], v["wo"], v["x"], v["e"]])


@pytest.mark.parametrize("sizes", [(20, 30, 4, 2, 16), (1, 40, 4, 4, 32), (140, 150, 2, 1, 80)])
@pytest.mark.parametrize("kind", sorted(KINDS))
def test_gradients_are_those_of_the_keep_all_executor(kind, sizes, ctx):
    f, nodes = attention_step(*sizes)
    want = [o.copy() for o in ad.Executor(nodes, ctx=ctx).run(f, convert_to_numpy_ret_vals=True)]
    ex = KINDS[kind](nodes, ctx=ctx)
    for _ in range(2):
        got = ex.run(f, convert_to_numpy_ret_vals=True)
        # the same operators: products of up to 64 terms in another order, 64 * 2^-24, through scores of up to some ten
        assert all(off(a, b) <= 1e-4 for a, b in zip(got, want)), [off(a, b) for a, b in zip(got, want)]


def step_of_the_model(cls, ctx, **kw):
    """What each parameter moves by in two steps."""
    m = transformer(vocab_size=60, d_model=32, num_heads=4, d_ff=48, num_blocks=1, maxlen1=9, maxlen2=8, batch_size=4, seed=11,
                    scaled_embedding=True, cross_attention=True)
    first = {v.name: np.array(v.tensor_value) for v in m.variables}
    f = m.synthetic_batch(4)
    for b in range(4):
        f[m.xs][b, 9 - 2 * b:] = 0
        f[m.ys_in][b, 7 - b:] = 0
    opt = optimizer.SGDOptimizer(0.05, ctx=ctx)
    rows = 4 * 7
    loss = ad.mul_byconst_op(ad.reduce_sum_op(ad.slice_op(m.token_scores(), (0, 0), (rows, 1)), [0, 1]), -1.0 / rows)
    train = opt.minimize(loss)
    ex = cls([loss, train], ctx=ctx, **kw)
    for _ in range(2):
        ex.run(f)
    now = {v.name: v.tensor_value for v in m.variables}
    return {n: (v.asnumpy() if isinstance(v, ndarray.NDArray) else np.asarray(v)) - first[n] for n, v in now.items()}


@pytest.mark.parametrize("kind", sorted(KINDS))
def test_parameters_move_as_under_the_keep_all_executor(kind, ctx):
    want, got = step_of_the_model(ad.Executor, ctx), step_of_the_model(KINDS[kind], ctx)
    assert {"dec0_cross_q_weight", "dec0_cross_kv_weight"} <= set(want)
    for name in want:
        # (a key's bias moves no score against another: what it moves by is rounding)
        if not np.linalg.norm(want[name]) or name.endswith("_k_bias"):
            continue
        assert off(got[name], want[name]) <= 1e-2, name

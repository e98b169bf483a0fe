"""The rows' log-sum-exps, which a cross attention's forward pass leaves for its gradients: whose they are, and that nobody takes
another pass's."""
import numpy as np
import pytest

from tsplit_b200 import ndarray, gpu_ops as ad


def graph():
    v = {k: ad.Variable(k) for k in ("q", "kv", "key", "g")}
    y = ad.cross_attention_op(v["q"], v["kv"], v["key"])
    return v, y, ad.cross_attention_gradient_op(y, v["g"])


def feeds(v, seed, n=2, tq=20, tk=30, h=2, d=16):
    r = np.random.default_rng(seed)
    return {v["q"]: r.standard_normal((n, tq, h, d), np.float32), v["kv"]: r.standard_normal((n, tk, 2, h, d), np.float32),
            v["key"]: np.ones((n, tk), np.float32), v["g"]: r.standard_normal((n, tq, h, d), np.float32)}


# ------------------------------------------------------------------------------------------------ a result that is fed
def test_a_fed_result_is_refused_where_the_step_is_planned():
    """The kernels' gradients need the forward pass in their own step; the NumPy path computes everything from its inputs."""
    v, y, grads = graph()
    f = feeds(v, 1)
    shapes = {n: a.shape for n, a in f.items()}
    ex = ad.Executor(grads)
    assert len(ex.run({**f, y: ad.Executor([y]).run(f)[0]})) == 2
    ex.on_device = True
    ex.infer_shape(shapes)
    with pytest.raises(ValueError, match="fed"):
        ex.infer_shape({**shapes, y: f[v["q"]].shape})
    only = ad.Executor([y])
    only.on_device = True
    only.infer_shape({**shapes, y: f[v["q"]].shape})                 # (nobody asks for a gradient)


@pytest.mark.gpu
@pytest.mark.parametrize("cls", [ad.Executor, ad.recomputeExecutor, ad.microopExecutor])
def test_a_fed_result_is_refused_whatever_ran_before(cls):
    """Forward passes over two batches, then gradients with the first one's result fed: its log-sum-exps are gone."""
    ctx = ndarray.gpu(0)
    v, y, grads = graph()
    forward = ad.Executor([y], ctx=ctx)
    first = forward.run(feeds(v, 1), convert_to_numpy_ret_vals=True)[0].copy()
    forward.run(feeds(v, 2))
    ex = cls([y] + grads, ctx=ctx)
    want = [ex.run(feeds(v, k), convert_to_numpy_ret_vals=True) for k in (1, 2)]
    for _ in range(2):
        for e in (ex, cls(grads, ctx=ctx)):
            with pytest.raises(ValueError, match="fed"):
                e.run({**feeds(v, 1), y: first})
    got = ex.run(feeds(v, 2), convert_to_numpy_ret_vals=True)
    assert all(np.array_equal(a, b) for a, b in zip(got, want[1]))


@pytest.mark.gpu
@pytest.mark.parametrize("cls", [ad.recomputeExecutor, ad.microopExecutor])
def test_operators_are_timed_one_by_one(cls):
    """Each node several times on its own, as a measured plan wants it; the same results afterwards."""
    ctx = ndarray.gpu(0)
    v, y, grads = graph()
    ex = cls([y] + grads, ctx=ctx)
    times = ex.measure_ops(feeds(v, 1))                # (before a plan that cuts operators in pieces)
    want = ad.Executor([y] + grads, ctx=ctx).run(feeds(v, 1), convert_to_numpy_ret_vals=True)
    assert {y, grads[0], grads[1], grads[0].inputs[0]} <= set(times) and all(t > 0 for t in times.values())
    assert all(np.array_equal(a, b) for a, b in zip(want, ex.run(feeds(v, 1), convert_to_numpy_ret_vals=True)))

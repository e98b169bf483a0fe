"""The rows' log-sum-exps, which a cross attention's forward pass leaves for its gradients: whose they are, and that nobody takes
another pass's."""
import gc

import numpy as np
import pytest
import torch

from tsplit_b200 import ndarray, gpu_ops as ad
from tsplit_b200.ops import _gpu as G, attention as A
from tsplit_b200.stream import Stream, create_stream_handle


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


# ------------------------------------------------------------------------------------------------ two streams
def test_every_stream_has_log_sum_exps_of_its_own():
    """... which are given back once neither the stream nor what was captured on it is there."""
    ctx, sizes = ndarray.cpu(0), (2, 20, 30, 2, 2, 16)
    _, y, _ = graph()
    a, b = Stream(ctx), Stream(ctx)
    assert A._row_sums(y, sizes, ctx, a, make=False) is None
    one, two = A._row_sums(y, sizes, ctx, a), A._row_sums(y, sizes, ctx, b)
    assert one.ptr != two.ptr
    assert A._row_sums(y, sizes, ctx, a) is one and A._row_sums(y, sizes, ctx, b, make=False) is two
    assert A._row_sums(y, sizes[:1] + (200,) + sizes[2:], ctx, a) is not one and A._row_sums(y, sizes, ctx, a) is one
    captured = a.buffers                                             # (as a captured graph holds it)
    del a
    gc.collect()
    A._row_sums(y, sizes, ctx, Stream(ctx))
    held = [x for x in y.state.values() if isinstance(x, ndarray.NDArray)]
    assert any(x is one for x in held) and len(held) == 4
    del captured, held
    gc.collect()
    three = Stream(ctx)
    new = A._row_sums(y, sizes, ctx, three)
    held = [x for x in y.state.values() if isinstance(x, ndarray.NDArray)]
    assert len(held) == 2 and any(x is two for x in held) and any(x is new for x in held)


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", [dict(), dict(tq=1, h=4), dict(tq=150, tk=200, d=128)])
def test_another_streams_forward_pass_in_between(sizes):
    """Two executors of the same nodes: one's forward pass stands between the other's and its gradients."""
    ctx = ndarray.gpu(0)
    v, y, grads = graph()
    f = [feeds(v, k, **sizes) for k in (1, 2)]
    want = [ad.Executor([y] + grads, ctx=ctx).run(x, convert_to_numpy_ret_vals=True) for x in f]
    st = [create_stream_handle(ctx) for _ in f]
    arr = [{n: ndarray.array(a, ctx, channels_last=False) for n, a in x.items()} for x in f]
    out = [{n: ndarray.empty(w.shape, ctx, channels_last=False) for n, w in zip([y] + grads, ws)} for ws in want]
    pre = grads[0].inputs[0]
    flat = ndarray.empty(pre.op.infer_shape(pre, [out[0][y].shape] * 2 + [arr[0][i].shape for i in y.inputs]), ctx)

    def run(k, n):
        vals = {**arr[k], **out[k], pre: flat}
        n.op.gpu_compute(n, [vals[i] for i in n.inputs], vals[n], st[k])
        st[k].sync()
    for k, n in ((0, y), (1, y), (0, pre), (0, grads[0]), (0, grads[1]), (1, pre), (1, grads[0]), (1, grads[1])):
        run(k, n)
    for o, w in zip(out, want):
        for n, a in zip([y] + grads, w):
            assert np.array_equal(o[n].asnumpy(), a)


# ------------------------------------------------------------------------------------------------ their room
@pytest.mark.parametrize("tq,shape", [(3, (2, 4, 3)), (3, (2, 4, 127)), (129, (2, 4, 129)), (129, (2, 4, 255)), (1, (2, 3, 128))])
def test_too_few_log_sum_exps_are_refused(tq, shape):
    """The kernels write and read them for whole tiles of 128 queries, so an array of as many as there are queries is too short."""
    e, sizes = ndarray.empty, (2, tq, 5, 4, 2, 8)
    q, kv, lse, flat = e((2, tq, 4, 8)), e((2, 5, 2, 2, 8)), e(shape), e((A._prepared_floats(*sizes),))
    for call in [lambda: G.cross_attention(q, kv, None, q, lse, sizes, 1.0, None),
                 lambda: G.cross_attention(q, kv, None, q, lse, sizes, 1.0, None, flat),
                 lambda: G.cross_attention_grad_q(flat, None, lse, q, sizes, 1.0, None),
                 lambda: G.cross_attention_grad_kv(flat, None, lse, kv, sizes, 1.0, None),
                 lambda: G.cross_attention_grads(flat, None, lse, q, kv, sizes, 1.0, None)]:
        with pytest.raises(ValueError, match="log-sum-exps"):
            call()


# ------------------------------------------------------------------------------------------------ launches
@pytest.mark.gpu
def test_launches_are_counted():
    """Every entry's count against the kernels that a capture of it holds: never more, and the same where no size decides."""
    from cuda.bindings import runtime as cudart
    from tsplit_b200.utils import launch_counter
    ctx = ndarray.gpu(0)
    st, e = create_stream_handle(ctx), lambda *s: ndarray.empty(s, ctx, channels_last=False)
    sizes = (2, 20, 30, 2, 2, 16)
    q, kv, key, y, dq, dkv, lse, flat = (e(2, 20, 2, 16), e(2, 30, 2, 2, 16), e(2, 30), e(2, 20, 2, 16), e(2, 20, 2, 16), e(2, 30, 2, 2, 16),
                                         e(2, 2, 128), e(A._prepared_floats(*sizes)))
    table, ids, rows = e(50, 16), e(600), e(600, 16)
    x, of_rows, out, g, dx = e(20, 100), e(20), e(20, 5), e(20, 5), e(20, 100)

    def real(call):
        def ok(r):
            assert int(r[0]) == 0
            return r[1] if len(r) > 1 else None
        call()                                                     # (scratch is there)
        st.sync()
        ok(cudart.cudaStreamBeginCapture(st.handle, cudart.cudaStreamCaptureMode.cudaStreamCaptureModeThreadLocal))
        before = launch_counter.count()
        call()
        counted = launch_counter.count() - before
        captured = ok(cudart.cudaStreamEndCapture(st.handle))
        r = cudart.cudaGraphGetNodes(captured)
        r = cudart.cudaGraphGetNodes(captured, r[-1])
        kernels = sum(ok(cudart.cudaGraphNodeGetType(n)) == cudart.cudaGraphNodeType.cudaGraphNodeTypeKernel for n in r[1])
        ok(cudart.cudaGraphDestroy(captured))
        return counted, kernels
    for a in (q, kv, y, lse, flat, x, out, g, rows, table):
        a.t.zero_()
    for a in (key, ids, of_rows):
        a.t.fill_(1.0)
    torch.cuda.synchronize()
    for call in [lambda: G.cross_attention(q, kv, key, y, lse, sizes, 1.0, st, flat), lambda: G.cross_attention_prepare_g(q, y, flat, sizes, st),
                 lambda: G.cross_attention_prepare(q, kv, key, q, y, flat, sizes, 1.0, st), lambda: G.cross_attention_grad_q(flat, key, lse, dq, sizes, 1.0, st),
                 lambda: G.cross_attention_grad_kv(flat, key, lse, dkv, sizes, 1.0, st),
                 lambda: G.cross_attention_grads(flat, key, lse, dq, dkv, sizes, 1.0, st), lambda: G.scaled_embedding(table, ids, rows, 1.0, st),
                 lambda: G.token_score(x, of_rows, out, 1, st), lambda: G.token_score_grad(x, of_rows, out, g, dx, st)]:
        counted, kernels = real(call)
        assert counted == kernels
    for call in [lambda: G.cross_attention(q, kv, key, y, lse, sizes, 1.0, st), lambda: G.scaled_embedding_grad(rows, ids, table, 1.0, None, st)]:
        counted, kernels = real(call)
        assert 1 <= counted <= kernels


@pytest.mark.gpu
@pytest.mark.parametrize("n,tq,tk,h,s,d", [(2, 200, 300, 4, 2, 64), (1, 129, 130, 3, 1, 80), (3, 9, 1, 1, 1, 8), (2, 1, 300, 4, 4, 64)])
def test_what_a_forward_pass_takes_outside_of_the_step(n, tq, tk, h, s, d):
    import ctypes
    from tsplit_b200 import _base
    ctx = ndarray.gpu(0)
    v, y, _ = graph()
    f = feeds(v, 1, n=n, tq=tq, tk=tk, h=h, d=d)
    f[v["kv"]] = np.ascontiguousarray(f[v["kv"]][:, :, :, :s])
    handle, held = ctypes.c_void_p(), _base.kernels().tsb_scratch_bytes
    held.restype = ctypes.c_longlong
    assert int(torch.cuda.cudart().cudaStreamCreate(ctypes.addressof(handle))) == 0        # (torch's streams come from a pool)
    ex = ad.StreamExecutor([y], ctx=ctx, stream=Stream(ctx, torch_stream=torch.cuda.ExternalStream(handle.value)))
    gc.collect()
    torch.cuda.synchronize()
    _base.kernels().tsb_scratch_trim()                               # (given-back buffers would be taken)
    before = held()
    ex.run(f)
    rows = sum(a.nbytes for a in y.state.values() if isinstance(a, ndarray.NDArray))
    assert rows + held() - before == y.op.workspace_bytes(y, [f[i].shape for i in y.inputs], f[v["q"]].shape)


def test_single_tokens_are_the_same_to_the_plan_and_to_the_kernels():
    import os
    import re
    source = open(os.path.join(os.path.dirname(A.__file__), "..", "csrc", "kernels", "cross_attention.cu")).read()
    assert int(re.search(r"\bFEW_ROWS = (\d+)", source).group(1)) == A.FEW_ROWS
    assert [A.keeps_operands((1, t, 4, 8), (1, 9, 2, 2, 8)) for t in (3, 4, 5)] == [False, False, True]

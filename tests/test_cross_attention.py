"""Attention across to an encoder's states: the NumPy path and the kernels against the definition in 64 bits, at lengths,
head layouts and masks where they can go wrong."""
import numpy as np
import pytest

from tsplit_b200 import ndarray, gpu_ops as ad

#: a pair of fp16 pieces keeps a number to 2^-22, the product of the low pieces that is left out is another 2^-22
PIECE = 2.0 ** -22
#: fp16 ends at 2^-25 (half of its last step): of a tile whose largest number is at least 2^13, of dS whose bound
#: |g| |v| + max|dot| (of the longest rows) is at least 2^14, of P whose 1 is 2^14
TILE, LAST = 2.0 ** -38, 2.0 ** -39


@pytest.fixture(params=[pytest.param("cpu"), pytest.param("gpu", marks=pytest.mark.gpu)])
def ctx(request):
    return None if request.param == "cpu" else ndarray.gpu(0)


def definition(q, kv, key, scale, g):
    """(y, dq, dkv) and bounds of what pieces of 2^-22 and fp32 sums may be off, element by element."""
    n, tq, h, d = q.shape
    tk, s = kv.shape[1], kv.shape[3]
    out = [np.zeros(a.shape) for a in (q, q, kv)]
    tol = [np.zeros(a.shape) for a in (q, q, kv)]
    for b in range(n):
        kept = np.arange(tk) if key is None else np.flatnonzero(key[b] != 0)
        if not len(kept):
            continue
        for j in range(h):
            t = j // (h // s)
            qq, k, v, gg = (a.astype(np.float64) for a in (q[b, :, j], kv[b, kept, 0, t], kv[b, kept, 1, t], g[b, :, j]))
            x = qq @ k.T * scale
            p = np.exp(x - x.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            y = p @ v
            dp, dot = gg @ v.T, (gg * y).sum(1, keepdims=True)
            ds = p * (dp - dot) * scale
            out[0][b, :, j], out[1][b, :, j] = y, ds @ k
            out[2][b, kept, 0, t] += ds.T @ qq
            out[2][b, kept, 1, t] += p.T @ gg
            # a product is off by three times PIECE of the sum of its terms' sizes (either factor, what is left out), and
            # by a truncation a step of its sum; a score's error e makes p off by a factor of e (its normaliser by no more)
            step = 3 * PIECE + d * 2.0 ** -23
            aq, ak, av, ag = (np.abs(a).max(initial=0) for a in (qq, k, v, gg))
            e = (np.abs(qq) @ np.abs(k).T * abs(scale)) * step + 2.0 ** -22 * (4 + np.abs(x))
            e += abs(scale) * TILE * (aq * np.abs(k).sum(1)[None, :] + ak * np.abs(qq).sum(1)[:, None])
            rel = 2 * e.max(1, keepdims=True) + len(kept) * 2.0 ** -24
            long = 3 * PIECE + 100 * 2.0 ** -23                   # 24 steps a tile, and up to 80 tiles
            dy = rel * (p @ np.abs(v)) + long * (p @ np.abs(v)) + LAST * np.abs(v).sum(0) + TILE * av
            tol[0][b, :, j] = dy
            ddp = np.abs(gg) @ np.abs(v).T * step + TILE * (ag * np.abs(v).sum(1)[None, :] + av * np.abs(gg).sum(1)[:, None])
            ddot = (np.abs(gg) * dy).sum(1, keepdims=True) + d * 2.0 ** -23 * (np.abs(gg) * np.abs(y)).sum(1, keepdims=True)
            dds = abs(scale) * p * (ddp + ddot) + rel * np.abs(ds) + abs(scale) * LAST * (1.1 * np.sqrt((gg ** 2).sum(1).max(initial=0) * (v ** 2).sum(1).max()) + np.abs(dot).max(initial=0))
            tol[1][b, :, j] = dds @ np.abs(k) + long * (np.abs(ds) @ np.abs(k)) + TILE * ak * np.abs(ds).sum(1, keepdims=True)
            tol[2][b, kept, 0, t] += dds.T @ np.abs(qq) + long * (np.abs(ds).T @ np.abs(qq)) + TILE * aq * np.abs(ds).sum(0)[:, None]
            tol[2][b, kept, 1, t] += (rel * p + LAST).T @ np.abs(gg) + long * (p.T @ np.abs(gg)) + TILE * ag * p.sum(0)[:, None]
    return out, tol


def graph(masked, scale):
    def build():
        q, kv, key, g = (ad.Variable(v) for v in ("q", "kv", "key", "g"))
        y = ad.cross_attention_op(q, kv, key if masked else None, scale=scale)
        names = {"q": q, "kv": kv, "g": g}
        if masked:
            names["key"] = key
        return names, [y] + ad.cross_attention_gradient_op(y, g)
    return build


def evaluate(build, feeds, ctx, **kw):
    names, nodes = build()
    ex = ad.Executor(nodes, ctx=ctx, **kw)
    return [np.asarray(o).astype(np.float64) for o in ex.run({names[k]: v for k, v in feeds.items()}, convert_to_numpy_ret_vals=True)]


def case(n, tq, tk, h, s, d, mask="tail", seed=0, spread=1.0):
    r = np.random.default_rng([n, tq, tk, h, s, d, seed])
    f = {"q": r.standard_normal((n, tq, h, d), np.float32) * np.float32(spread), "kv": r.standard_normal((n, tk, 2, s, d), np.float32),
         "g": r.standard_normal((n, tq, h, d), np.float32)}
    if mask:
        key = r.integers(1, 9, (n, tk)).astype(np.float32)
        if mask == "tail":                                        # the last sentence is padding all through
            for b in range(n):
                key[b, tk - tk * b // max(1, n - 1):] = 0
        elif mask == "holes":
            key[r.random((n, tk)) < 0.6] = 0
        elif mask == "head":
            key[:, :tk - 1] = 0
        f["key"] = key
    return f


def check(f, ctx, scale=None, **kw):
    got = evaluate(graph("key" in f, scale), f, ctx, **kw)
    want, tol = definition(f["q"], f["kv"], f.get("key"), scale if scale is not None else f["q"].shape[3] ** -0.5, f["g"])
    for name, a, b, t in zip(("y", "dq", "dkv"), got, want, tol):
        assert a.shape == b.shape and np.isfinite(a).all(), name
        worst = np.unravel_index(np.argmax(np.abs(a - b) - t), a.shape)
        assert np.all(np.abs(a - b) <= t + 1e-37), "%s at %s: %r for %r, tolerance %r" % (name, worst, a[worst], b[worst], t[worst])
        assert not a[t == 0].any(), name                           # what is masked has no result and no gradient at all
    return got


@pytest.mark.parametrize("n,tq,tk,h,s,d", [(1, 1, 1, 1, 1, 1), (2, 1, 5, 2, 2, 8), (2, 3, 40, 4, 2, 32), (1, 8, 130, 2, 2, 64), (2, 9, 33, 2, 2, 64),
                                           (3, 30, 37, 4, 4, 32), (1, 128, 128, 1, 1, 64), (2, 129, 127, 2, 1, 64), (1, 70, 300, 3, 1, 20),
                                           (2, 17, 129, 2, 2, 128), (1, 140, 260, 2, 1, 100), (1, 33, 65, 2, 2, 69), (1, 20, 64, 1, 1, 3)])
@pytest.mark.parametrize("mask", [None, "tail", "holes", "head"])
def test_attention_and_its_gradients(n, tq, tk, h, s, d, mask, ctx):
    check(case(n, tq, tk, h, s, d, mask), ctx)


@pytest.mark.gpu
@pytest.mark.parametrize("n,tq,tk,h,s,d", [(4, 255, 256, 8, 8, 64), (1, 600, 1100, 4, 1, 64), (1, 500, 1030, 4, 2, 128), (2, 1, 3000, 8, 2, 128),
                                           (1, 2, 5000, 4, 1, 64), (70, 1, 40, 2, 2, 32), (3, 385, 513, 2, 2, 96), (1, 1300, 200, 2, 1, 64),
                                           (5, 10, 700, 1, 1, 128)])
@pytest.mark.parametrize("mask", [None, "tail", "holes"])
def test_longer_attention(n, tq, tk, h, s, d, mask):
    check(case(n, tq, tk, h, s, d, mask), ndarray.gpu(0))


@pytest.mark.parametrize("tq", [1, 40])
@pytest.mark.parametrize("spread,scale", [(8.0, None), (1.0, 0.0), (1.0, -0.3), (3.0, 1.0)])
def test_attention_scales_and_peaks(tq, spread, scale, ctx):
    check(case(2, tq, 150, 2, 1, 64, "holes", spread=spread), ctx, scale=scale)


@pytest.mark.parametrize("tq", [1, 150])
@pytest.mark.parametrize("sizes", [(1e-3, 1e-6, 1e-12), (1e-20, 1e18, 1e-9), (30.0, 3e5, 1e20), (1.0, 1e-30, 1e30)])
def test_attention_of_small_and_large_numbers(tq, sizes, ctx):
    """Queries, states and gradients far from 1: pieces of 16 bits have to be scaled."""
    f = case(2, tq, 260, 2, 1, 64, "holes")
    for k, v in zip(("q", "kv", "g"), sizes):
        f[k] = f[k] * np.float32(v)
    check(f, ctx, scale=1.0 / (8 * sizes[0] * sizes[1]))


@pytest.mark.parametrize("tq", [1, 150])
def test_attention_of_rows_of_unequal_size(tq, ctx):
    """Rows whose sizes differ by up to 2^12, side by side in a tile."""
    f = case(2, tq, 300, 4, 2, 64, "holes")
    r = np.random.default_rng(2)
    for k in ("q", "kv", "g"):
        f[k] *= 2.0 ** -r.integers(0, 13, f[k].shape[:2] + (1,) * (f[k].ndim - 2)).astype(np.float32)
    check(f, ctx)


@pytest.mark.parametrize("tq", [1, 33])
@pytest.mark.parametrize("what", [np.nan, np.inf, np.finfo(np.float32).max])
def test_what_masked_states_hold_does_not_matter(tq, what, ctx):
    f = case(3, tq, 200, 2, 2, 64, "holes")
    f["key"][1] = 0
    clean = [a.copy() for a in check(f, ctx)]
    f["kv"][f["key"] == 0] = what
    for a, b in zip(evaluate(graph(True, None), f, ctx), clean):
        assert np.array_equal(a, b)


@pytest.mark.parametrize("tq", [1, 4, 33, 200])
@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf])
def test_a_query_that_is_no_number_stays_alone(tq, what, ctx):
    """Its own row is NaN, and through it its head's states; other rows, heads and sentences keep their results to the bit."""
    f = case(2, tq, 150, 4, 2, 64, "holes")
    clean = check(f, ctx)
    f["q"][1, tq // 2, 2, 5] = what
    y, dq, dkv = evaluate(graph(True, None), f, ctx)
    rows = np.zeros(y.shape, bool)
    rows[1, tq // 2, 2] = True
    states = np.zeros(dkv.shape, bool)
    states[1, f["key"][1] != 0, :, 1] = True
    for got, was, bad in ((y, clean[0], rows), (dq, clean[1], rows), (dkv, clean[2], states)):
        assert np.isnan(got[bad]).all() and np.array_equal(got[~bad], was[~bad])


@pytest.mark.parametrize("tq", [1, 4, 33, 200])
@pytest.mark.parametrize("which", [0, 1])
def test_a_state_that_is_no_number_shows(tq, which, ctx):
    """Every query that reads it is NaN (with a NaN value: in its column at least); no other head's or sentence's is."""
    f = case(2, tq, 150, 4, 2, 64, "holes")
    clean = check(f, ctx)
    f["key"][1, 70] = 1
    f["kv"][1, 70, which, 1, 9] = np.nan
    y = evaluate(graph(True, None), f, ctx)[0]
    assert np.isnan(y[1, :, 2:, 9]).all() and (which or np.isnan(y[1, :, 2:]).all())
    assert np.array_equal(y[0], clean[0][0])
    f["key"][1, 70] = 0
    assert np.isfinite(evaluate(graph(True, None), f, ctx)[0]).all()


@pytest.mark.parametrize("n,tq,tk", [(0, 4, 5), (2, 0, 5), (2, 4, 0), (2, 20, 0)])
def test_empty_attention(n, tq, tk, ctx):
    y, dq, dkv = evaluate(graph(True, None), case(n, tq, tk, 2, 2, 16, None) | {"key": np.ones((n, tk), np.float32)}, ctx)
    assert y.shape == dq.shape == (n, tq, 2, 16) and dkv.shape == (n, tk, 2, 2, 16)
    assert not y.any() and not dq.any() and not dkv.any()


def test_gradients_by_differences():
    """The NumPy gradients against central differences of the definition."""
    f = case(2, 3, 7, 4, 2, 5, "holes")
    f["key"][0] = 1
    _, dq, dkv = evaluate(graph(True, 0.7), f, None)
    def loss(**kw):
        a = {**f, **kw}
        return (definition(a["q"], a["kv"], a["key"], 0.7, a["g"])[0][0] * a["g"]).sum()
    h = 1e-5
    for name, got in (("q", dq), ("kv", dkv)):
        for at in list(np.ndindex(*got.shape))[::7]:
            up, down = f[name].astype(np.float64), f[name].astype(np.float64)
            up[at] += h
            down[at] -= h
            assert abs((loss(**{name: up}) - loss(**{name: down})) / (2 * h) - got[at]) <= 1e-5


def test_attention_in_a_training_graph(ctx):
    """Projections around it, and every gradient through ``ad.gradients``, against the same from separate operators."""
    n, tq, tk, h, d = 2, 11, 9, 2, 16
    r = np.random.default_rng(3)
    feeds = {"x": r.standard_normal((n * tq, 8), np.float32), "e": r.standard_normal((n * tk, 8), np.float32),
             "wq": r.standard_normal((8, h * d), np.float32) * 0.3, "wkv": r.standard_normal((8, 2 * h * d), np.float32) * 0.3,
             "key": (np.arange(n * tk).reshape(n, tk) % 4).astype(np.float32), "w": r.standard_normal((n, tq, h, d), np.float32)}

    def build(fused):
        def make():
            v = {k: ad.Variable(k) for k in feeds}
            q = ad.array_reshape_op(ad.matmul_op(v["x"], v["wq"]), (n, tq, h, d))
            kv = ad.array_reshape_op(ad.matmul_op(v["e"], v["wkv"]), (n, tk, 2, h, d))
            if fused:
                y = ad.cross_attention_op(q, kv, v["key"])
            else:
                flat = ad.matmul_op(v["e"], v["wkv"])
                k, val = (ad.array_reshape_op(ad.slice_op(flat, (0, i * h * d), (n * tk, h * d)), (n, tk, h, d)) for i in (0, 1))
                p = ad.masked_softmax_op(ad.batch_matmul_op(q, k, trans_B=True, heads_A=True, heads_B=True), v["key"], scale=d ** -0.5)
                y = ad.batch_matmul_op(p, val, heads_B=True, heads_out=True)
            loss = ad.reduce_sum_op(ad.mul_op(y, v["w"]), [0, 1, 2, 3])
            return v, [y] + ad.gradients(loss, [v["wq"], v["wkv"], v["x"], v["e"]])
        return make
    one, parts = evaluate(build(True), feeds, ctx), evaluate(build(False), feeds, None)
    for a, b in zip(one, parts):
        # the projections around it take ten bits of each factor on the GPU
        assert np.allclose(a, b, rtol=0, atol=(2e-5 if ctx is None else 0.02) * np.abs(b).max())


def test_attention_refuses(ctx):
    shapes = {"q": (2, 3, 4, 8), "kv": (2, 5, 2, 2, 8), "key": (2, 5), "g": (2, 3, 4, 8)}
    for change in [{"q": (2, 3, 32)}, {"kv": (2, 5, 2, 8)}, {"kv": (2, 5, 3, 2, 8)}, {"kv": (1, 5, 2, 2, 8)}, {"kv": (2, 5, 2, 3, 8)},
                   {"kv": (2, 5, 2, 2, 4)}, {"key": (2, 4)}, {"g": (2, 3, 4, 4)}, {"q": (2, 3, 4, 129), "kv": (2, 5, 2, 2, 129), "g": (2, 3, 4, 129)}]:
        with pytest.raises(AssertionError):
            evaluate(graph(True, None), {k: np.ones(v, np.float32) for k, v in {**shapes, **change}.items()}, ctx)


def test_attention_refuses_what_is_not_row_major():
    import torch
    from tsplit_b200.ops import _gpu as G
    cpu = ndarray.cpu(0)
    q = ndarray.NDArray(torch.zeros(2, 8, 4, 3).permute(0, 3, 2, 1), cpu)                 # (2, 3, 4, 8)
    ok, kv, rows, flat = ndarray.empty((2, 3, 4, 8)), ndarray.empty((2, 5, 2, 2, 8)), ndarray.empty((2, 4, 3)), ndarray.empty((64,))
    sizes = (2, 3, 5, 4, 2, 8)
    for call in [lambda: G.cross_attention(q, kv, None, ok, rows, sizes, 1.0, None),
                 lambda: G.cross_attention_prepare(ok, kv, None, q, ok, flat, sizes, 1.0, None),
                 lambda: G.cross_attention_grad_q(flat, None, rows, q, sizes, 1.0, None),
                 lambda: G.cross_attention_grad_kv(flat, None, q, kv, sizes, 1.0, None)]:
        with pytest.raises(ValueError, match="row-major"):
            call()


@pytest.mark.gpu
def test_attention_has_the_same_bits_every_time_in_a_captured_step():
    """Replays of one graph, another executor's in between on its own stream."""
    a, b = case(2, 150, 300, 4, 2, 64, "holes"), case(3, 1, 900, 4, 4, 128, "holes")
    first, ex = {}, {}
    for k, f in (("a", a), ("b", b)):
        names, nodes = graph(True, None)()
        ex[k] = (ad.Executor(nodes, ctx=ndarray.gpu(0), use_graph=True), {names[x]: v for x, v in f.items()})
    for _ in range(5):
        for k in ("a", "b"):
            got = ex[k][0].run(ex[k][1], convert_to_numpy_ret_vals=True)
            if k not in first:
                first[k] = [x.copy() for x in got]
            for x, y in zip(got, first[k]):
                assert np.array_equal(x, y)


@pytest.mark.gpu
@pytest.mark.parametrize("tq", [1, 20])
def test_attention_of_arrays_that_begin_anywhere(tq):
    """Arrays 4 bytes off a 16-byte boundary take the loads of single numbers, with the same results."""
    import torch
    from tsplit_b200.ops import _gpu as G, attention as A
    from tsplit_b200.stream import create_stream_handle
    ctx = ndarray.gpu(0)
    st = create_stream_handle(ctx)
    f = case(2, tq, 100, 2, 1, 64, "holes")
    sizes, got = (2, tq, 100, 2, 1, 64), []
    for off in (0, 1):
        def at(v):
            t = torch.empty(v.size + 8, device="cuda")[off:off + v.size].view(v.shape)
            return ndarray.from_tensor(t.copy_(torch.from_numpy(v)), ctx)
        q, kv, key, g = (at(f[k]) for k in ("q", "kv", "key", "g"))
        y, dq, dkv, lse = at(f["q"] * 0), at(f["q"] * 0), at(f["kv"] * 0), ndarray.empty((2, 2, 128), ctx, use_pool=False)
        flat = ndarray.empty((A._prepared_floats(*sizes),), ctx, use_pool=False)
        torch.cuda.synchronize()
        G.cross_attention(q, kv, key, y, lse, sizes, 0.125, st)
        G.cross_attention_prepare(q, kv, key, g, y, flat, sizes, 0.125, st)
        G.cross_attention_grad_q(flat, key, lse, dq, sizes, 0.125, st)
        G.cross_attention_grad_kv(flat, key, lse, dkv, sizes, 0.125, st)
        st.sync()
        got.append([a.asnumpy() for a in (y, dq, dkv)])
    want, tol = definition(f["q"], f["kv"], f["key"], 0.125, f["g"])
    for a, b, w, t in zip(got[0], got[1], want, tol):
        assert np.all(np.abs(a - w) <= t + 1e-37) and np.all(np.abs(b - w) <= t + 1e-37)


def test_room_for_the_gradients_operands_is_checked():
    """A flat array that is too short, or off a 16-byte boundary, is refused before anything is launched."""
    import ctypes
    from tsplit_b200 import _base
    from tsplit_b200.ops import attention as A
    if not _base.have("libtsplit_kernels.so"):
        pytest.skip("the kernel library is not built")
    lib = _base._load("libtsplit_kernels.so")
    sizes = (2, 3, 5, 4, 2, 8)
    some, need, p, i, f = ctypes.c_void_p(1 << 20), 4 * A._prepared_floats(*sizes), ctypes.c_void_p, ctypes.c_int, ctypes.c_float
    for at, have in [(1 << 20, need - 16), (0, need), ((1 << 20) + 4, need)]:
        at, have, rest = p(at), ctypes.c_int64(have), [i(s) for s in sizes] + [f(1.0), p(0)]
        assert lib.tsb_cross_attention_prepare(some, some, p(0), some, some, at, have, *rest) == 1
        assert lib.tsb_cross_attention_grad_q(at, have, p(0), some, some, *rest) == 1
        assert lib.tsb_cross_attention_grad_kv(at, have, p(0), some, some, *rest) == 1
    for bad in [(2, 3, 5, 4, 3, 8), (2, 3, 5, 4, 2, 129), (2, 3, 5, 4, 2, 0), (-1, 3, 5, 4, 2, 8), (2, 3, 5, 0, 2, 8)]:
        assert lib.tsb_cross_attention(some, some, p(0), some, some, *[i(s) for s in bad], f(1.0), p(0)) == 1


@pytest.mark.gpu
def test_a_result_that_was_fed_has_no_gradient():
    """The kernels of the gradients read the log-sum-exps of the forward pass, which did not run on these queries."""
    ctx, f = ndarray.gpu(0), case(2, 20, 30, 2, 2, 16, None)
    names, nodes = graph(False, None)()
    first = [np.asarray(o) for o in ad.Executor(nodes, ctx=ctx).run({names[k]: v for k, v in f.items()}, convert_to_numpy_ret_vals=True)]
    feeds = {names["q"]: f["q"] * 2, names["kv"]: f["kv"], names["g"]: f["g"], nodes[0]: first[0]}
    with pytest.raises(ValueError):
        ad.Executor(nodes[1:], ctx=ctx).run(feeds)
    again = ad.Executor(nodes, ctx=ctx).run({names[k]: v for k, v in f.items()}, convert_to_numpy_ret_vals=True)
    assert all(np.array_equal(a, np.asarray(b)) for a, b in zip(first, again))


@pytest.mark.gpu
def test_states_that_grow_take_no_more_room():
    """A decoder's states grow by one a step: the node keeps one array of log-sum-exps for all of them."""
    ctx = ndarray.gpu(0)
    q, kv, g = (ad.Variable(v) for v in ("q", "kv", "g"))
    y = ad.cross_attention_op(q, kv)
    ex = ad.Executor([y] + ad.cross_attention_gradient_op(y, g), ctx=ctx)
    for tk in (5, 6, 7, 130):
        f = case(2, 1, tk, 4, 2, 32, None)
        got = [np.asarray(o, np.float64) for o in ex.run({q: f["q"], kv: f["kv"], g: f["g"]}, convert_to_numpy_ret_vals=True)]
        want, tol = definition(f["q"], f["kv"], None, 32 ** -0.5, f["g"])
        assert all(np.all(np.abs(a - b) <= t) for a, b, t in zip(got, want, tol))
    assert sum(isinstance(v, ndarray.NDArray) for v in y.state.values()) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("n,tq,tk,h,s,d", [(2, 300, 700, 4, 2, 64), (1, 200, 400, 2, 2, 128), (8, 2000, 20, 8, 8, 64), (2, 10, 5000, 2, 2, 64), (1, 5, 6, 1, 1, 3),
                                           (4, 900, 1000, 16, 16, 32)])
def test_both_gradients_in_one_call_in_a_captured_chain(n, tq, tk, h, s, d):
    """Many blocks and few ones of either kernel, beside one another: the bits of two calls, and whoever reads the first
    gradient right behind the second finds it done."""
    import torch
    from tsplit_b200.ops import _gpu as G
    from tsplit_b200.ops.attention import _prepared_floats
    from tsplit_b200.runtime import cudagraph
    from tsplit_b200.stream import create_stream_handle
    ctx = ndarray.gpu(0)
    st, sizes = create_stream_handle(ctx), (n, tq, tk, h, s, d)
    f = {k: torch.from_numpy(v).cuda() for k, v in case(n, tq, tk, h, s, d, "holes").items()}
    y, dq, dq2, seen = (torch.zeros_like(f["q"]) for _ in range(4))
    dkv, dkv2, seen2 = (torch.zeros_like(f["kv"]) for _ in range(3))
    lse = torch.zeros(n, h, -(-tq // 128) * 128, device="cuda")
    prepared = torch.zeros(_prepared_floats(*sizes), device="cuda")
    q, kv, key, g, Y, DQ, DQ2, S, DKV, DKV2, S2, L, P = (ndarray.from_tensor(t, ctx) for t in (
        f["q"], f["kv"], f["key"], f["g"], y, dq, dq2, seen, dkv, dkv2, seen2, lse, prepared))
    torch.cuda.synchronize()
    G.cross_attention(q, kv, key, Y, L, sizes, 0.3, st)
    G.cross_attention_prepare(q, kv, key, g, Y, P, sizes, 0.3, st)
    G.cross_attention_grad_q(P, key, L, DQ, sizes, 0.3, st)
    G.cross_attention_grad_kv(P, key, L, DKV, sizes, 0.3, st)

    def step():
        for _ in range(3):
            for a in (P, L, DQ2, DKV2):
                G.fill(a, 0.0, st)
            G.cross_attention(q, kv, key, Y, L, sizes, 0.3, st)
            G.cross_attention_prepare(q, kv, key, g, Y, P, sizes, 0.3, st)
            G.cross_attention_grads(P, key, L, DQ2, DKV2, sizes, 0.3, st)
            G.unary(G.UN_MULC, DQ2, S, st, alpha=1.0)
            G.unary(G.UN_MULC, DKV2, S2, st, alpha=1.0)
    step()
    st.sync()
    captured = cudagraph.capture(st, step)
    for _ in range(20):
        captured.launch(st)
        st.sync()
        assert torch.equal(seen, dq) and torch.equal(seen2, dkv)


@pytest.mark.gpu
@pytest.mark.parametrize("tq,heads,kept", [(9, 2, True), (8, 2, False), (3, 8, True), (40, 2, True)])
def test_a_step_splits_its_operands_once(tq, heads, kept):
    """The pieces of q, k and v that the forward pass makes are those of the gradients, but for single tokens, which make none;
    both gradients go in one call; a second gradient of the same node takes operands of its own."""
    ctx, f = ndarray.gpu(0), case(2, tq, 70, heads, 2, 16, "holes")
    v = {k: ad.Variable(k) for k in f}
    y = ad.cross_attention_op(v["q"], v["kv"], v["key"])
    nodes = [y] + ad.cross_attention_gradient_op(y, v["g"])
    want, tol = definition(f["q"], f["kv"], f["key"], 0.25, f["g"])
    for more in (False, True):
        if more:
            nodes = nodes + ad.cross_attention_gradient_op(y, ad.mul_byconst_op(v["g"], 2.0))
        ex = ad.Executor(nodes, ctx=ctx)
        for _ in range(2):
            got = [np.asarray(o, np.float64) for o in ex.run({v[k]: a for k, a in f.items()}, convert_to_numpy_ret_vals=True)]
        for a, b, t in zip(got, want, tol):
            assert np.all(np.abs(a - b) <= t + 1e-37)
        for a, b, t in zip(got[3:], want[1:], tol[1:]):
            assert np.all(np.abs(a - 2 * b) <= 2 * t + 1e-37)
        kinds = [what for what, _ in ex._step_plan.actions]
        assert kinds.count("keep") == (2 if kept and not more else 0) and kinds.count("attention") == (2 if more else 1)

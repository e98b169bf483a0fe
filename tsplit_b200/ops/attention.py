"""Attention across to an encoder's states, as one operator with its gradients.

The reference's example builds it from batched products, a scale, a padding mask and a soft-max
(``examples/transformer.py:117-171``) and keeps the scores; here they never leave the chip
(``csrc/kernels/cross_attention.cu``), forward or backward.

On the GPU a number takes part in the products to 2^-22 of itself or 2^-38 of the largest number in its tile, 128 rows of a head of
the queries, keys, values or gradients, whichever is more, and a probability to 2^-39; sums are fp32.  So results have the accuracy of
fp32 where the rows of a tile are within 2^16 of one another, and a row that is smaller loses some of its own (its gradient is off by
1e-5 of itself where another row's is 2^20 times as large, by 1 % at 2^30).  The forward pass of up to eight rows of queries to a head
of the states is plain fp32.
"""
from __future__ import annotations

import weakref

import numpy as np

from ..graph import Op
from ..stream import Buffers
from . import _gpu as G

MAX_HEAD_DIM = 128


def _sizes(q, kv, key=None):
    """(N, Tq, Tk, heads, heads of the states, d) of shapes that belong together."""
    assert len(q) == 4 and len(kv) == 5 and kv[2] == 2, \
        "queries are [N, Tq, heads, d] and states [N, Tk, 2, heads, d], not %s and %s" % (tuple(q), tuple(kv))
    n, tq, h, d = q
    assert kv[0] == n and kv[4] == d and kv[3] > 0 and h % kv[3] == 0, "queries %s do not fit states %s" % (tuple(q), tuple(kv))
    assert 0 < d <= MAX_HEAD_DIM, "a head has 1 to %d columns, not %d" % (MAX_HEAD_DIM, d)
    assert key is None or tuple(key) == (n, kv[1]), "key tokens are [N, Tk] = %s, not %s" % ((n, kv[1]), tuple(key))
    return n, tq, kv[1], h, kv[3], d


def _heads(x, shared):
    """[N, T, heads, d] -> [N, shared, heads / shared, T, d] in 64 bits."""
    n, t, h, d = x.shape
    return x.astype(np.float64).reshape(n, t, shared, h // shared, d).transpose(0, 2, 3, 1, 4)


def _back(x):
    n, s, r, t, d = x.shape
    return x.transpose(0, 3, 1, 2, 4).reshape(n, t, s * r, d)


def _probabilities(q, kv, key, scale):
    """(P, q, k, v) in 64 bits, a row without keys all zero; what is masked is taken out whatever it holds."""
    s = kv.shape[3]
    k, v = _heads(kv[:, :, 0], s), _heads(kv[:, :, 1], s)
    q = _heads(q, s)
    keep = np.ones((kv.shape[0], kv.shape[1]), bool) if key is None else key != 0
    at = keep[:, None, None, :, None]
    k, v = np.where(at, k, 0), np.where(at, v, 0)
    with np.errstate(invalid="ignore"):                     # (a query that is no number)
        x = np.where(keep[:, None, None, None, :], q @ np.swapaxes(k, 3, 4) * scale, -np.inf)
        m = x.max(axis=4, keepdims=True, initial=-np.inf)
        p = np.exp(x - np.where(np.isneginf(m), 0, m))
    z = p.sum(axis=4, keepdims=True)
    return p / np.where(z == 0, 1, z), q, k, v


class CrossAttentionOp(Op):
    """``softmax(scale * q k^T) v`` of queries [N, Tq, heads, d] over an encoder's states [N, Tk, 2, shared, d], keys and values
    of one projection; ``heads / shared`` consecutive query heads read each head of the states.  ``key_tokens`` [N, Tk]: states
    whose token is 0 are padding and take no part, whatever they hold; a query that has none left gives 0 and no gradient.
    ``scale`` defaults to ``d ** -0.5``.  Up to eight queries of a head of the states (single tokens) take a path of their own."""
    name = "CrossAttention"

    def __call__(self, q, kv, key_tokens=None, scale=None):
        node = Op.__call__(self, *([q, kv] + ([key_tokens] if key_tokens is not None else [])),
                           scale=None if scale is None else float(scale))
        node.state = {}
        return node

    @staticmethod
    def scale_of(node, d):
        return node.attrs["scale"] if node.attrs["scale"] is not None else float(d) ** -0.5

    def np_compute(self, node, iv):
        p, _, _, v = _probabilities(iv[0], iv[1], iv[2] if len(iv) > 2 else None, self.scale_of(node, iv[0].shape[3]))
        return _back(p @ v).astype(np.float32)

    def gpu_compute(self, node, iv, out, stream, prepared=None):
        sizes = _sizes(iv[0].shape, iv[1].shape, iv[2].shape if len(iv) > 2 else None)
        G.cross_attention(iv[0], iv[1], iv[2] if len(iv) > 2 else None, out, _row_sums(node, sizes, iv[0].ctx, stream), sizes,
                          self.scale_of(node, sizes[5]), stream, prepared)

    def gradient(self, node, g):
        return cross_attention_gradient_op(node, g) + [None] * (len(node.inputs) - 2)

    def infer_shape(self, node, s):
        _sizes(s[0], s[1], s[2] if len(s) > 2 else None)
        return tuple(s[0])

    def flops(self, node, s, out):
        return 4.0 * np.prod(s[0]) * s[1][1]

    def workspace_bytes(self, node, s, out):
        """The pieces of the operands, scratch of the stream outside any pool (where a step plan keeps them for the gradients, they lie
        in an array of the step instead); and the log-sum-exps."""
        n, tq, tk, h, shared, d = _sizes(s[0], s[1])
        rows = 4 * n * h * _whole_tiles(tq)
        if not keeps_operands(s[0], s[1]):
            return rows
        q, k = n * h * _whole_tiles(tq) // 128, n * shared * _whole_tiles(tk) // 128
        return rows + 4 * _prepared_floats(n, tq, tk, h, shared, d) - q * (128 * (64 if d <= 64 else 128) * 4 + 2 * 128 * 4) - -(-q // 2) * 16


_NO_STREAM = Buffers()


def _row_sums(node, sizes, ctx, stream, make=True):
    """The rows' log-sum-exps, which the forward kernel leaves for the gradients.  An array for every stream, since two executors of
    one node may run at once or in turn, for as long as the stream or what was captured on it lives; and for every number of rows that
    was run there, since a step that was captured at one goes on using its own (a sentence of states that grows needs no more)."""
    shape = (sizes[0], sizes[3], _whole_tiles(sizes[1]))
    held = stream.buffers if stream is not None else _NO_STREAM        # (one object for all that is launched on a stream)
    key, owners = ("lse", shape, ctx, id(held)), node.state.setdefault("owners", {})
    owner = owners.get(key)
    if owner is not None and owner() is held:
        return node.state[key]
    if not make:
        return None
    for k, o in list(owners.items()):
        if o() is None:
            owners.pop(k, None)
            node.state.pop(k, None)
    from .. import ndarray
    node.state[key] = ndarray.empty(shape, ctx, use_pool=False)
    owners[key] = weakref.ref(held)
    return node.state[key]


def _whole_tiles(t):
    return -(-t // 128) * 128


def _prepared_floats(n, tq, tk, h, shared, d):
    """Length of what the gradients read: tiles of 128 rows and 64 or 128 columns of q, k, v and g, two numbers for each, and
    two for every row of g."""
    q, k, columns = n * h * _whole_tiles(tq) // 128, n * shared * _whole_tiles(tk) // 128, 64 if d <= 64 else 128
    return 128 * columns * 2 * (q + k) + 2 * (-(-q // 2) * 4 + -(-k // 2) * 4) + 2 * 128 * q


class CrossAttentionPrepareOp(Op):
    """Operands of both gradients as the tensor cores take them, and ``sum(g * y)`` over every row: a flat array that only the
    kernels read.  The gradients also read what the forward kernel has left, so it has to run in the same step: where its result
    is fed, the step is refused as it is planned (the NumPy path computes everything from its inputs)."""
    name = "CrossAttentionPrepare"

    def __call__(self, g, forward):
        return Op.__call__(self, g, forward, *forward.inputs, scale=forward.attrs["scale"], fwd=forward)

    def np_compute(self, node, iv):
        return np.zeros(self.infer_shape(node, [v.shape for v in iv]), np.float32)

    def gpu_compute(self, node, iv, out, stream, kept=False):
        """``kept``: the forward pass of this step has left the pieces of its operands in ``out``."""
        g, y, q, kv = iv[:4]
        key = iv[4] if len(iv) > 4 else None
        sizes = _sizes(q.shape, kv.shape, key.shape if key is not None else None)
        if kept:
            G.cross_attention_prepare_g(g, y, out, sizes, stream)
            return
        G.cross_attention_prepare(q, kv, key, g, y, out, sizes, CrossAttentionOp.scale_of(node, sizes[5]), stream)

    def gradient(self, node, g):
        raise NotImplementedError

    def check_feeds(self, node, fed):
        if node.attrs["fwd"] in fed:
            raise ValueError("the gradient of a cross attention takes the forward pass of the same step, not a result that was fed")

    def infer_shape(self, node, s):
        assert tuple(s[0]) == tuple(s[1]) == tuple(s[2]), "gradient %s of a result %s" % (tuple(s[0]), tuple(s[1]))
        return (_prepared_floats(*_sizes(s[2], s[3], s[4] if len(s) > 4 else None)),)

    def flops(self, node, s, out):
        return 8.0 * np.prod(out)


class _CrossAttentionGradient(Op):
    def __call__(self, prepared, g, forward):
        return Op.__call__(self, prepared, g, *forward.inputs, scale=forward.attrs["scale"], fwd=forward)

    def _ds(self, node, iv):
        g, q, kv, key = iv[1], iv[2], iv[3], iv[4] if len(iv) > 4 else None
        p, q, k, v = _probabilities(q, kv, key, CrossAttentionOp.scale_of(node, q.shape[3]))
        g = _heads(g, kv.shape[3])
        dp = g @ np.swapaxes(v, 3, 4)
        ds = p * (dp - (dp * p).sum(4, keepdims=True)) * CrossAttentionOp.scale_of(node, kv.shape[4])
        return ds, p, g, q, k

    @staticmethod
    def _arguments(node, iv, ctx, stream):
        """(prepared, key tokens, log-sum-exps), sizes, scale."""
        key = iv[4] if len(iv) > 4 else None
        sizes = _sizes(iv[2].shape, iv[3].shape, key.shape if key is not None else None)
        lse = _row_sums(node.attrs["fwd"], sizes, ctx, stream, make=False)
        assert lse is not None, "the gradient of a cross attention needs its forward pass on the same stream first"
        return (iv[0], key, lse), sizes, CrossAttentionOp.scale_of(node, sizes[5])

    def gpu_compute(self, node, iv, out, stream):
        inputs, sizes, scale = self._arguments(node, iv, out.ctx, stream)
        self._launch(*inputs, out, sizes, scale, stream)

    def gradient(self, node, g):
        raise NotImplementedError

    def _check(self, s):
        sizes = _sizes(s[2], s[3], s[4] if len(s) > 4 else None)
        assert tuple(s[1]) == tuple(s[2]) and tuple(s[0]) == (_prepared_floats(*sizes),), \
            "gradient %s of a result %s" % (tuple(s[1]), tuple(s[2]))


class CrossAttentionGradQueryOp(_CrossAttentionGradient):
    name = "CrossAttentionGradQuery"
    _launch = staticmethod(G.cross_attention_grad_q)

    def np_compute(self, node, iv):
        ds, _, _, _, k = self._ds(node, iv)
        return _back(ds @ k).astype(np.float32)

    def infer_shape(self, node, s):
        self._check(s)
        return tuple(s[2])

    def flops(self, node, s, out):
        return 6.0 * np.prod(s[2]) * s[3][1]


class CrossAttentionGradStatesOp(_CrossAttentionGradient):
    name = "CrossAttentionGradStates"
    _launch = staticmethod(G.cross_attention_grad_kv)

    def np_compute(self, node, iv):
        ds, p, g, q, _ = self._ds(node, iv)
        dk, dv = ((np.swapaxes(a, 3, 4) @ b).sum(2, keepdims=True) for a, b in ((ds, q), (p, g)))
        both = np.stack([_back(dk), _back(dv)], 2).astype(np.float32)
        if len(iv) > 4:                                        # (also where a query that is no number meets them)
            both[iv[4] == 0] = 0
        return both

    def infer_shape(self, node, s):
        self._check(s)
        return tuple(s[3])

    def flops(self, node, s, out):
        return 8.0 * np.prod(s[2]) * s[3][1]


#: rows of queries to a head of the states up to which the forward pass takes the path for single tokens (the kernels' constant of
#: that name; where they keep operands for such rows, they refuse)
FEW_ROWS = 8


def keeps_operands(q, kv):
    """Whether the forward pass over these shapes splits its operands: all but single tokens do."""
    return q[2] // kv[3] * q[1] > FEW_ROWS


def both_gradients(nodes, iv, out, stream):
    """The gradients of the queries and of the states (``nodes``, of one forward pass and one set of operands ``iv``) into the
    arrays ``out``, in one call."""
    inputs, sizes, scale = nodes[0].op._arguments(nodes[0], iv, out[0].ctx, stream)
    G.cross_attention_grads(*inputs, *out, sizes, scale, stream)


_ca, _cap, _cagq, _cagkv = CrossAttentionOp(), CrossAttentionPrepareOp(), CrossAttentionGradQueryOp(), CrossAttentionGradStatesOp()


def cross_attention_op(q, kv, key_tokens=None, scale=None):
    return _ca(q, kv, key_tokens, scale)


def cross_attention_gradient_op(node, g):
    """[gradient of the queries, gradient of the states] of a :func:`cross_attention_op` ``node`` whose result has ``g``."""
    prepared = _cap(g, node)
    return [_cagq(prepared, g, node), _cagkv(prepared, g, node)]

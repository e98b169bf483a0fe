"""Softmax and softmax cross-entropy.

Capability parity: ``gpu_ops/Softmax.py:6-60`` and
``gpu_ops/SoftmaxCrossEntropy.py:39-118``.  The reference kernels run
``<<<1,1024>>>`` with one thread per row and a serial mean
(``src/ops/Softmax.cu:3-22``, ``SoftmaxCrossEntropy.cu:5-104``); here each row is
reduced by one warp (or one CTA for wide rows) across all SMs and the mean is a
deterministic two-stage reduction.
"""
from __future__ import annotations

import numpy as np

from ..graph import Op
from . import _gpu as G


def softmax_func(y):
    b = y - np.max(y, axis=-1, keepdims=True)
    e = np.exp(b)
    return e / np.sum(e, axis=-1, keepdims=True)


class SoftmaxOp(Op):
    name = "Softmax"

    def __call__(self, x):
        return Op.__call__(self, x)

    def np_compute(self, node, iv):
        return softmax_func(iv[0]).astype(np.float32)

    def cpu_compute(self, node, iv, out):
        from .. import cpu_links
        if not cpu_links.ok(iv[0], out):
            return False
        cpu_links.softmax(iv[0], out)
        return True

    def gpu_compute(self, node, iv, out, stream):
        G.softmax(iv[0], out, stream)

    def gradient(self, node, g):
        # the reference leaves this undefined (src/ops/Softmax.cu has no backward kernel)
        return [softmax_gradient_op(node, g)]

    def infer_shape(self, node, s):
        return tuple(s[0])

    def flops(self, node, s, out):
        return 5.0 * np.prod(out)


class SoftmaxGradientOp(Op):
    """``dx = y * (dy - sum(dy * y, axis=-1, keepdims=True))`` in one kernel (y and dy read once)."""
    name = "SoftmaxGradient"

    def __call__(self, y, dy):
        return Op.__call__(self, y, dy)

    def np_compute(self, node, iv):
        y, dy = iv
        return (y * (dy - np.sum(dy * y, axis=-1, keepdims=True))).astype(np.float32)

    def cpu_compute(self, node, iv, out):
        from .. import cpu_links
        if not cpu_links.ok(iv[0], iv[1], out):
            return False
        cpu_links.softmax_grad(iv[0], iv[1], out)
        return True

    def gpu_compute(self, node, iv, out, stream):
        G.softmax_grad(iv[0], iv[1], out, stream)

    def gradient(self, node, g):
        raise NotImplementedError

    def infer_shape(self, node, s):
        assert tuple(s[0]) == tuple(s[1])
        return tuple(s[0])

    def flops(self, node, s, out):
        return 4.0 * np.prod(out)


class MaskedSoftmaxOp(Op):
    """Attention soft-max in one kernel: ``softmax(scale * scores + mask)`` over the last axis of
    ``scores [N, H, Tq, Tk]``.  ``key_tokens [N, Tk]`` (optional second input): keys whose token id is 0 are
    padding and get -1e9 added; ``causal``: keys behind the query (j > q) are replaced by -1e9.  Equals the chain
    the reference's example builds from separate operators (``examples/transformer.py:139-158``: scale, padding
    mask through a broadcast add, causal ``where``, soft-max), without their passes over the score tensor."""
    name = "MaskedSoftmax"

    def __call__(self, scores, key_tokens=None, scale=1.0, causal=False):
        ins = [scores] + ([key_tokens] if key_tokens is not None else [])
        return Op.__call__(self, *ins, scale=float(scale), causal=bool(causal))

    def np_compute(self, node, iv):
        x = iv[0].astype(np.float32) * np.float32(node.attrs["scale"])
        if len(iv) > 1:
            pad = (iv[1] == 0).astype(np.float32) * np.float32(-1e9)
            x = x + pad.reshape(pad.shape[0], 1, 1, pad.shape[-1])
        if node.attrs["causal"]:
            tq, tk = x.shape[-2], x.shape[-1]
            future = np.arange(tk)[None, :] > np.arange(tq)[:, None]
            x = np.where(future, np.float32(-1e9), x)
        return softmax_func(x).astype(np.float32)

    def gpu_compute(self, node, iv, out, stream):
        x = iv[0]
        assert x.is_contiguous() and out.is_contiguous() and len(x.shape) == 4
        key = iv[1] if len(iv) > 1 else None
        G.masked_softmax(x, key, out, node.attrs["scale"], node.attrs["causal"], stream)

    def gradient(self, node, g):
        grads = [masked_softmax_gradient_op(node, g, node.attrs["scale"])]
        if len(node.inputs) > 1:
            from .misc import zeroslike_op
            grads.append(zeroslike_op(node.inputs[1]))
        return grads

    def infer_shape(self, node, s):
        assert len(s[0]) == 4, "scores are [N, H, Tq, Tk]"
        if len(s) > 1:
            assert tuple(s[1]) == (s[0][0], s[0][3]), "key tokens are [N, Tk]"
        return tuple(s[0])

    def flops(self, node, s, out):
        return 7.0 * np.prod(out)


class MaskedSoftmaxGradientOp(Op):
    """``dx = scale * y * (dy - sum(dy * y, axis=-1, keepdims=True))`` (masked positions have y = 0)."""
    name = "MaskedSoftmaxGradient"

    def __call__(self, y, dy, scale=1.0):
        return Op.__call__(self, y, dy, scale=float(scale))

    def np_compute(self, node, iv):
        y, dy = iv
        return (np.float32(node.attrs["scale"]) * y * (dy - np.sum(dy * y, axis=-1, keepdims=True))).astype(np.float32)

    def gpu_compute(self, node, iv, out, stream):
        G.scaled_softmax_grad(iv[0], iv[1], out, node.attrs["scale"], stream)

    def gradient(self, node, g):
        raise NotImplementedError

    def infer_shape(self, node, s):
        assert tuple(s[0]) == tuple(s[1])
        return tuple(s[0])

    def flops(self, node, s, out):
        return 5.0 * np.prod(out)


class SoftmaxCrossEntropyOp(Op):
    """``mean_rows(-sum(labels * log softmax(logits)))`` -> shape (1,)."""
    name = "SoftmaxCrossEntropy"

    def __call__(self, logits, labels):
        return Op.__call__(self, logits, labels)

    def np_compute(self, node, iv):
        y, y_ = iv
        b = y - np.max(y, axis=1, keepdims=True)
        logsm = b - np.log(np.sum(np.exp(b), axis=1, keepdims=True))
        return np.mean(-np.sum(y_ * logsm, axis=1), keepdims=True).astype(np.float32)

    def gpu_compute(self, node, iv, out, stream):
        G.softmax_ce(iv[0], iv[1], out, stream)

    def cpu_compute(self, node, iv, out):
        from .. import cpu_links
        if not cpu_links.ok(iv[0], iv[1], out):
            return False
        cpu_links.softmax_crossentropy(iv[0], iv[1], out)
        return True

    def gradient(self, node, g):
        from .misc import zeroslike_op
        return [softmaxcrossentropy_gradient_op(node.inputs[0], node.inputs[1], g),
                zeroslike_op(node.inputs[1])]

    def infer_shape(self, node, s):
        assert tuple(s[0]) == tuple(s[1]), "logits %s and labels %s differ" % (s[0], s[1])
        return (1,)

    def flops(self, node, s, out):
        return 6.0 * np.prod(s[0])


class SoftmaxCrossEntropyGradientOp(Op):
    """``(softmax(logits) - labels) * g / rows``."""
    name = "SoftmaxCrossEntropyGradient"

    def __call__(self, logits, labels, g):
        return Op.__call__(self, logits, labels, g)

    def np_compute(self, node, iv):
        y, y_, g = iv
        return ((softmax_func(y) - y_) * g.reshape(-1)[0] / y.shape[0]).astype(np.float32)

    def cpu_compute(self, node, iv, out):
        from .. import cpu_links
        if not cpu_links.ok(iv[0], iv[1], iv[2], out) or iv[0].ndim != 2 or iv[2].size != 1:
            return False
        cpu_links.softmax_crossentropy_grad(iv[0], iv[1], iv[2], out)
        return True

    def gpu_compute(self, node, iv, out, stream):
        G.softmax_ce_grad(iv[0], iv[1], iv[2], out, stream)

    def gradient(self, node, g):
        raise NotImplementedError

    def infer_shape(self, node, s):
        return tuple(s[0])

    def flops(self, node, s, out):
        return 6.0 * np.prod(out)


MAX_ALTERNATIVES = 32


class TokenLogProbOp(Op):
    """What a language model says about given tokens, from one pass over its ``logits`` [rows, vocab]: a row of
    ``3 + 2 * top_k`` numbers

        log p(id), entropy of p, log-sum-exp of the logits, log p of the ``top_k`` likeliest tokens (falling), their ids

    with p the soft-max of the row.  ``ids``: one whole number a row, in any shape; one outside [0, vocab) means no token and
    gives 0.  Logits of -inf are tokens that cannot be said.  A row that has no other logit has log-sum-exp and log
    probabilities of -inf, no entropy and no gradient.  Of equal logits the one with the lower id comes first; a NaN makes its
    row's numbers NaN and is not among the likeliest (id -1 where fewer than ``top_k`` logits are numbers).  Gradients reach
    the logits from every column but the ids."""
    name = "TokenLogProb"

    def __call__(self, logits, ids, top_k=0):
        top_k = int(top_k)
        assert 0 <= top_k <= MAX_ALTERNATIVES, "top_k is 0 to %d, not %d" % (MAX_ALTERNATIVES, top_k)
        return Op.__call__(self, logits, ids, top_k=top_k)

    def np_compute(self, node, iv):
        x, top = iv[0].astype(np.float64), node.attrs["top_k"]
        ids = iv[1].reshape(-1).astype(np.int64)
        with np.errstate(invalid="ignore", divide="ignore"):
            m = x.max(1, keepdims=True)
            empty = (x == -np.inf).all(1)
            u = x - np.where(empty[:, None], 0, m)
            e = np.exp(u)
            z = e.sum(1)
            lse = np.where(empty, 0, m[:, 0]) + np.log(z)
            h = np.log(z) - np.where(e == 0, 0, e * u).sum(1) / z
            out = np.empty((x.shape[0], 3 + 2 * top))
            given = (ids >= 0) & (ids < x.shape[1])
            own = x[np.arange(len(ids)), np.where(given, ids, 0)] - lse
            out[:, 0] = np.where(given, np.where(empty, -np.inf, own), 0)
            out[:, 1] = np.where(empty, 0, h)
            out[:, 2] = lse
            cols = np.argsort(-x, axis=1, kind="stable")[:, :top]          # (NaN last)
            best = np.take_along_axis(x, cols, 1)
            out[:, 3:3 + top] = np.where(empty[:, None], -np.inf, best - lse[:, None])
            out[:, 3 + top:] = np.where(np.isnan(best), -1, cols)
        return out.astype(np.float32)

    def gpu_compute(self, node, iv, out, stream):
        G.token_score(iv[0], iv[1], out, node.attrs["top_k"], stream)

    def gradient(self, node, g):
        return [token_log_prob_gradient_op(node.inputs[0], node.inputs[1], node, g), None]

    def infer_shape(self, node, s):
        assert len(s[0]) == 2 and np.prod(s[1], dtype=np.int64) == s[0][0], \
            "logits are [rows, vocab] with one id a row, not %s with %s" % (tuple(s[0]), tuple(s[1]))
        assert node.attrs["top_k"] <= s[0][1], "%d alternatives of %d tokens" % (node.attrs["top_k"], s[0][1])
        return (s[0][0], 3 + 2 * node.attrs["top_k"])

    def flops(self, node, s, out):
        return 8.0 * np.prod(s[0])


class TokenLogProbGradientOp(Op):
    """``sum_i w_i (1[c = id_i] - p_c) + w_lse p_c - w_H p_c (log p_c + H)``: w is the gradient ``g`` of a
    :class:`TokenLogProbOp`'s result ``out`` for these logits and ids, i its given token and the likeliest ones."""
    name = "TokenLogProbGradient"

    def __call__(self, logits, ids, out, g):
        return Op.__call__(self, logits, ids, out, g)

    def np_compute(self, node, iv):
        x, ids, out, g = iv[0].astype(np.float64), iv[1].reshape(-1).astype(np.int64), iv[2], iv[3].astype(np.float64)
        top, rows = (out.shape[1] - 3) // 2, np.arange(x.shape[0])
        with np.errstate(invalid="ignore"):
            m = x.max(1, keepdims=True)
            empty = (x == -np.inf).all(1)
            e = np.exp(x - np.where(empty[:, None], 0, m))
            z = np.where(empty, 1, e.sum(1))[:, None]
            p, logs = e / z, x - np.where(empty[:, None], 0, m) - np.log(z)
            h = -np.where(p == 0, 0, p * logs).sum(1, keepdims=True)
            dx = g[:, 2:3] * p - g[:, 1:2] * np.where(p == 0, 0, p * (logs + h))
            given = (ids >= 0) & (ids < x.shape[1])
            for j in range(top + 1):
                col = np.where(given, ids, -1) if j == 0 else out[:, 2 + top + j].astype(np.int64)
                w = np.where(col >= 0, g[:, 0] if j == 0 else g[:, 2 + j], 0)
                dx -= w[:, None] * p
                dx[rows, np.maximum(col, 0)] += w
            dx[empty] = 0
        return dx.astype(np.float32)

    def gpu_compute(self, node, iv, out, stream):
        G.token_score_grad(iv[0], iv[1], iv[2], iv[3], out, stream)

    def gradient(self, node, g):
        raise NotImplementedError

    def infer_shape(self, node, s):
        assert len(s[0]) == 2 and np.prod(s[1], dtype=np.int64) == s[0][0], \
            "logits are [rows, vocab] with one id a row, not %s with %s" % (tuple(s[0]), tuple(s[1]))
        assert tuple(s[2]) == tuple(s[3]) and len(s[2]) == 2 and s[2][0] == s[0][0] and s[2][1] >= 3 and s[2][1] % 2, \
            "results %s and gradients %s do not belong to logits %s" % (tuple(s[2]), tuple(s[3]), tuple(s[0]))
        return tuple(s[0])

    def flops(self, node, s, out):
        return 8.0 * np.prod(out)


_tlp, _tlpg = TokenLogProbOp(), TokenLogProbGradientOp()


def token_log_prob_op(logits, ids, top_k=0):
    return _tlp(logits, ids, top_k)


def token_log_prob_gradient_op(logits, ids, node, g):
    return _tlpg(logits, ids, node, g)


_sm, _ce, _ceg = SoftmaxOp(), SoftmaxCrossEntropyOp(), SoftmaxCrossEntropyGradientOp()
_smg = SoftmaxGradientOp()


def softmax_op(node):
    return _sm(node)


def softmax_gradient_op(node_y, node_dy):
    return _smg(node_y, node_dy)


_msm, _msmg = MaskedSoftmaxOp(), MaskedSoftmaxGradientOp()


def masked_softmax_op(scores, key_tokens=None, scale=1.0, causal=False):
    return _msm(scores, key_tokens, scale, causal)


def masked_softmax_gradient_op(node_y, node_dy, scale=1.0):
    return _msmg(node_y, node_dy, scale)


def softmaxcrossentropy_op(node_A, node_B):
    return _ce(node_A, node_B)


def softmaxcrossentropy_gradient_op(node_A, node_B, node_C):
    return _ceg(node_A, node_B, node_C)

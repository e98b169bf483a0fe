"""Operators around the attention stack of a language model, timed alone: tokens in (scaled embedding lookup and its
gradient by sorted tokens), attention across to an encoder's states (training and single-token steps), tokens out
(log probability of given tokens with entropy and top alternatives, and the gradient).

With ``own`` the calls go through the define-then-run API (``ad.*_op`` nodes, an executor that replays a CUDA graph) on
arrays that live on the GPU; without it the same values are computed by elementary torch operations in 32 bits.
``exact`` restates each operator from its definition in 64 bits.  Token ids are whole numbers held in fp32, the
framework's array type.
"""
import math
import zlib

import torch

own = False


# ---------------------------------------------------------------------------------------------------- the cases
def embed(tokens, vocab, dim, padded, **kw):
    return dict(kind="embed", tokens=tokens, vocab=vocab, dim=dim, padded=padded, **kw)


def score(rows, vocab, top, grad, **kw):
    return dict(kind="score", rows=rows, vocab=vocab, top=top, grad=grad, **kw)


def cross(n, tq, tk, heads, shared, dim, grad, **kw):
    """``shared``: heads of the keys and values, each read by ``heads / shared`` query heads."""
    return dict(kind="cross", n=n, tq=tq, tk=tk, heads=heads, shared=shared, dim=dim, grad=grad, **kw)


def listed():
    return [
        # one sentence of a few words over a small vocabulary: launches and latency
        embed(37, 500, 128, True, name="embed_sentence"),
        # odd everything: rows of no whole 16 bytes, ids of no round number
        embed(4099, 10007, 301, False, name="embed_odd"),
        # the Transformer example's batch: 32 sentences of 256 over 32000 words, 512 wide
        embed(8192, 32000, 512, True, name="embed_batch"),
        # a large batch over a large table: bound by memory
        embed(131072, 64000, 1024, True, name="embed_large"),
        # one row of logits while a sentence is written, five alternatives
        score(1, 32000, 5, False, name="score_token"),
        # ragged: odd vocabulary, values and gradient, eight alternatives
        score(1110, 10007, 8, True, name="score_ragged"),
        # the Transformer example's decoder positions: 32 x 255 rows over 32000 words, trained on
        score(8160, 32000, 0, True, name="score_train"),
        # prompt scoring over a large vocabulary, twenty alternatives
        score(4096, 128001, 20, False, name="score_prompt"),
        # a decoder's step: one query a sentence over 256 encoder states
        cross(32, 1, 256, 8, 8, 64, False, name="cross_step"),
        # the same over long documents, four query heads to each head of the cached states
        cross(4, 1, 16384, 16, 4, 128, False, name="cross_step_long"),
        # the Transformer example's decoder block in training
        cross(32, 255, 256, 8, 8, 64, True, name="cross_train"),
        # long documents in training, shared heads, lengths of no whole tile
        cross(2, 2000, 4111, 16, 4, 128, True, name="cross_long"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["embed", "score", "cross", "cross"])
    if kind == "embed":
        return embed(_log(rng, 1, 131072), _log(rng, 100, 64000), _log(rng, 8, 1024), rng.random() < 0.5)
    if kind == "score":
        vocab = _log(rng, 50, 128001)
        return score(_log(rng, 1, max(1, min(8192, 524000000 // vocab))), vocab, rng.choice([0, 1, 5, 8, 20, rng.randint(2, 32)]),
                     rng.random() < 0.5 and vocab < 64000)
    shared = rng.choice([1, 2, 4, 8])
    heads = shared * rng.choice([1, 1, 2, 4])
    dim = rng.choice([32, 64, 64, 128, 8 * rng.randint(1, 16), rng.randint(5, 128)])
    if rng.random() < 0.4:
        tk = _log(rng, 1, 16384)
        n = _log(rng, 1, max(1, min(64, 2000000000 // (8 * tk * shared * dim))))
        return cross(n, rng.choice([1, 1, 1, rng.randint(2, 5)]), tk, heads, shared, dim, False)
    n, tq, tk = _log(rng, 1, 32), _log(rng, 1, 2048), _log(rng, 1, 4200)
    n = max(1, min(n, 2 * 16 * 2000 * 4111 // (heads * tq * tk)))
    return cross(n, tq, tk, heads, shared, dim, rng.random() < 0.6)


# ---------------------------------------------------------------------------------------------------- the inputs
def _gen(name, seed):
    return torch.Generator(device="cuda").manual_seed((zlib.crc32(name.encode()) + 7919 * int(seed)) % (1 << 31))


def _normal(name, shape, seed):
    return torch.randn(tuple(shape), generator=_gen(name, seed), device="cuda")


def _uniform(name, shape, seed):
    return torch.rand(tuple(shape), generator=_gen(name, seed), device="cuda")


def _words(name, count, vocab, seed):
    """Token ids whose frequency falls with their number, as words of a text do."""
    u = _uniform(name, (count,), seed).double()
    return torch.exp(u * math.log(vocab)).floor().clamp_(1, vocab - 1)


def inputs(case, seed):
    """What a pass reads, by name."""
    k = case["kind"]
    if k == "embed":
        ids = _words("ids", case["tokens"], case["vocab"], seed)
        if case["padded"]:          # the tail of a sentence is padding, id 0
            ids = torch.where(_uniform("pad", ids.shape, seed) < 0.3, torch.zeros_like(ids), ids)
        return {"table": _normal("table", (case["vocab"], case["dim"]), seed) * case["dim"] ** -0.5, "ids": ids.float(),
                "g": _normal("g", (case["tokens"], case["dim"]), seed) * 1e-3}
    if k == "score":
        rows, vocab = case["rows"], case["vocab"]
        x = _normal("x", (rows, vocab), seed) * 2.5
        if vocab > 64:              # words that may not be said, as constrained decoding masks them
            x[:, 7::97] = float("-inf")
        ids = torch.randint(0, vocab, (rows,), generator=_gen("ids", seed), device="cuda")
        ids = torch.where(ids % 97 == 7, ids - 1, ids)
        ids[::19] = -1              # positions without a token
        if rows == 1:
            ids = ids.abs()
        got = {"x": x, "ids": ids.float()}
        if case["grad"]:
            w = torch.full((3 + 2 * case["top"],), 0.05, device="cuda")
            w[0], w[1], w[2] = -1.0, -0.01, 1e-3
            got["g"] = _normal("g", (rows, w.numel()), seed).abs_() * w / rows
        return got
    n, tq, tk, h, s, d = (case[v] for v in ("n", "tq", "tk", "heads", "shared", "dim"))
    ends = torch.randint((tk + 1) // 2, tk + 1, (n, 1), generator=_gen("len", seed), device="cuda")
    ends[0] = tk
    if n > 4:
        ends[4] = 0                 # a sentence that is padding all through
    word = torch.randint(1, 32000, (n, tk), generator=_gen("key", seed), device="cuda").float()
    got = {"q": _normal("q", (n, tq, h, d), seed), "kv": _normal("kv", (n, tk, 2, s, d), seed),
           "key": torch.where(torch.arange(tk, device="cuda") < ends, word, torch.zeros_like(word))}
    if case["grad"]:
        got["g"] = _normal("g", (n, tq, h, d), seed) * 1e-3
    return got


def _embed_scale(case):
    return math.sqrt(case["dim"])


# ---------------------------------------------------------------------------------------------------- the calls
def prepare(case, seed):
    state = {"case": case, "in": inputs(case, seed)}
    if own:
        state["executor"], state["split"] = _build(case, state["in"])
    return state


def _build(case, given):
    """The executor that a user's program keeps, over arrays that are on the GPU already, and how its results are read."""
    from tsplit_b200 import gpu_ops as ad, ndarray
    ctx = ndarray.gpu(0)
    v = {k: ad.Variable(name=k, value=ndarray.from_tensor(t, ctx)) for k, t in given.items()}
    if case["kind"] == "embed":
        scale = _embed_scale(case)
        y = ad.scaled_embedding_op(v["table"], v["ids"], scale=scale, padding_id=0)
        nodes = [y, ad.scaled_embedding_gradient_op(v["g"], v["ids"], v["table"], scale=scale, padding_id=0)]
        names = ["y", "dtable"]
    elif case["kind"] == "score":
        y = ad.token_log_prob_op(v["x"], v["ids"], top_k=case["top"])
        nodes, names = [y], ["packed"]
        if case["grad"]:
            nodes.append(ad.token_log_prob_gradient_op(v["x"], v["ids"], y, v["g"]))
            names.append("dx")
    else:
        y = ad.cross_attention_op(v["q"], v["kv"], v["key"])
        nodes, names = [y], ["y"]
        if case["grad"]:
            nodes += ad.cross_attention_gradient_op(y, v["g"])
            names += ["dq", "dkv"]
    return ad.Executor(nodes, ctx=ctx, use_graph=True), names


def run(state):
    case = state["case"]
    if own:
        got = {k: o.t for k, o in zip(state["split"], state["executor"].run({}))}
        return _columns(got, case["top"]) if case["kind"] == "score" else got
    return {"embed": _plain_embed, "score": _plain_score, "cross": _plain_cross}[case["kind"]](case, state["in"])


def _columns(got, top):
    p = got.pop("packed")
    got.update(logp=p[:, 0], entropy=p[:, 1], lse=p[:, 2])
    if top:
        got.update(top=p[:, 3:3 + top], top_ids=p[:, 3 + top:])
    return got


# ---------------------------------------------------------------------------------------------------- plain forms
def _plain_embed(case, a):
    ids = a["ids"].long()
    y = a["table"][ids] * _embed_scale(case)
    g = torch.where((ids == 0)[:, None], torch.zeros((), device="cuda"), a["g"] * _embed_scale(case))
    return {"y": y, "dtable": torch.zeros_like(a["table"]).index_add_(0, ids, g)}


def _places(x, top):
    """Columns of the largest values of each row, ties by the lowest column."""
    bits = (x + 0.0).view(torch.int32)
    order = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long() * (1 << 32) - torch.arange(x.shape[1], device=x.device)
    return torch.topk(order, top, dim=1).indices


def _plain_score(case, a):
    x, ids, top = a["x"], a["ids"].long(), case["top"]
    given = ids >= 0
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    z = e.sum(1, keepdim=True)
    lse = m + torch.log(z)
    p = e / z
    logs = x - lse
    h = -torch.where(p > 0, p * logs, torch.zeros_like(p)).sum(1)
    at = ids.clamp(min=0)[:, None]
    got = {"logp": torch.where(given, logs.gather(1, at)[:, 0], torch.zeros_like(h)), "entropy": h, "lse": lse[:, 0]}
    cols = _places(x, top) if top else None
    if top:
        got.update(top=logs.gather(1, cols), top_ids=cols.float())
    if case["grad"]:
        g = a["g"]
        w = torch.where(given, g[:, 0], torch.zeros_like(h))
        total = g[:, 2] - w - g[:, 3:3 + top].sum(1)
        dx = p * (total[:, None] - g[:, 1:2] * torch.where(p > 0, logs + h[:, None], torch.zeros_like(p)))
        dx.scatter_add_(1, at, w[:, None])
        if top:
            dx.scatter_add_(1, cols, g[:, 3:3 + top])
        got["dx"] = dx
    return got


def _plain_cross(case, a):
    n, tq, tk, h, s, d = (case[v] for v in ("n", "tq", "tk", "heads", "shared", "dim"))
    scale = 1.0 / math.sqrt(d)

    def heads(t, count):            # [n, t, heads, d] -> [n, shared, heads / shared * t, d]
        return t.view(n, -1, s, count // s, d).permute(0, 2, 3, 1, 4).reshape(n, s, -1, d)
    q = heads(a["q"], h)
    k, v = heads(a["kv"][:, :, 0].contiguous(), s), heads(a["kv"][:, :, 1].contiguous(), s)
    keep = (a["key"] != 0).view(n, 1, 1, tk)
    x = torch.where(keep, torch.matmul(q, k.transpose(2, 3)) * scale, torch.full((), float("-inf"), device="cuda"))
    m = x.amax(3, keepdim=True)
    p = torch.where(keep, torch.exp(x - torch.where(m > float("-inf"), m, torch.zeros_like(m))), torch.zeros((), device="cuda"))
    p = p / p.sum(3, keepdim=True).clamp(min=1e-30)
    y = torch.matmul(p, v)

    def back(t, count):
        return t.view(n, s, count // s, -1, d).permute(0, 3, 1, 2, 4).reshape(n, -1, count, d)
    got = {"y": back(y, h)}
    if case["grad"]:
        g = heads(a["g"], h)
        ds = p * (torch.matmul(g, v.transpose(2, 3)) - (g * y).sum(3, keepdim=True)) * scale
        got["dq"] = back(torch.matmul(ds, k), h)
        got["dkv"] = torch.stack([back(torch.matmul(ds.transpose(2, 3), q), s), back(torch.matmul(p.transpose(2, 3), g), s)], 2)
    return got


# ---------------------------------------------------------------------------------------------------- the floor
def work(case):
    """Inputs read and outputs written once; flops of the products (the backward pass computes the scores again)."""
    k = case["kind"]
    if k == "embed":
        m, v, d = case["tokens"], case["vocab"], case["dim"]
        return {"bytes": 4.0 * (min(m, v) * d + m * d + 2 * m + m * d + v * d), "flops": 2.0 * m * d}
    if k == "score":
        x = case["rows"] * case["vocab"]
        return {"bytes": 4.0 * (x * (2 if case["grad"] else 1) + case["rows"] * (4 + 2 * case["top"])), "flops": 4.0 * x}
    n, tq, tk, h, s, d = (case[v] for v in ("n", "tq", "tk", "heads", "shared", "dim"))
    rows, states = n * tq * h * d, n * tk * 2 * s * d
    if not case["grad"]:
        return {"bytes": 4.0 * (2 * rows + states + n * tk), "flops": 4.0 * n * tq * tk * h * d}
    return {"bytes": 4.0 * (4 * rows + 2 * states + n * tk), "flops": 14.0 * n * tq * tk * h * d}


# ---------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    a = inputs(case, seed)
    if case["kind"] == "embed":
        ids, scale = a["ids"].long(), _embed_scale(case)
        dtable = torch.zeros((case["vocab"], case["dim"]), dtype=torch.float64, device="cuda")
        for i in range(0, case["tokens"], 32768):
            part = ids[i:i + 32768]
            word = part != 0
            dtable.index_add_(0, part[word], a["g"][i:i + 32768][word].double())
        return {"y": a["table"].double()[ids] * scale, "dtable": dtable * scale}
    if case["kind"] == "score":
        return _exact_score(case, a)
    return _exact_cross(case, a)


def _exact_score(case, a):
    top, parts = case["top"], []
    step = max(1, 40000000 // case["vocab"])
    for i in range(0, case["rows"], step):
        x, ids = a["x"][i:i + step].double(), a["ids"][i:i + step].long()
        r = torch.arange(x.shape[0], device="cuda")
        logs = torch.log_softmax(x, 1)
        p = logs.exp()
        h = torch.special.entr(p).sum(1)
        one = torch.zeros_like(p)
        one[r[ids >= 0], ids[ids >= 0]] = 1
        got = {"logp": torch.where(ids >= 0, logs[r, ids.clamp(min=0)], 0.0), "entropy": h, "lse": torch.logsumexp(x, 1)}
        if top:
            cols = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top]
            got.update(top=logs.gather(1, cols), top_ids=cols.double())
        if case["grad"]:
            g = a["g"][i:i + step].double()
            dx = g[:, :1] * (one - p * one.sum(1, keepdim=True)) + g[:, 2:3] * p
            dx -= g[:, 1:2] * torch.where(p > 0, p * (logs + h[:, None]), 0.0)
            for j in range(top):
                dx -= g[:, 3 + j:4 + j] * p
                dx[r, cols[:, j]] += g[:, 3 + j]
            got["dx"] = dx
        parts.append(got)
    return {k: torch.cat([v[k] for v in parts]) for k in parts[0]}


def _exact_cross(case, a):
    n, h, s, d = case["n"], case["heads"], case["shared"], case["dim"]
    per, scale = h // s, case["dim"] ** -0.5
    y = torch.zeros(a["q"].shape, dtype=torch.float64, device="cuda")
    dq, dkv = torch.zeros_like(y), torch.zeros(a["kv"].shape, dtype=torch.float64, device="cuda")
    for b in range(n):
        kept = a["key"][b].nonzero()[:, 0]
        if not kept.numel():
            continue
        for j in range(h):
            q, k, v = a["q"][b, :, j].double(), a["kv"][b, kept, 0, j // per].double(), a["kv"][b, kept, 1, j // per].double()
            p = torch.softmax(q @ k.T * scale, 1)
            y[b, :, j] = p @ v
            if case["grad"]:
                g = a["g"][b, :, j].double()
                dp = g @ v.T
                ds = p * (dp - (dp * p).sum(1, keepdim=True)) * scale
                dq[b, :, j] = ds @ k
                dkv[b, kept, 0, j // per] += ds.T @ q
                dkv[b, kept, 1, j // per] += p.T @ g
    return {"y": y, "dq": dq, "dkv": dkv} if case["grad"] else {"y": y}

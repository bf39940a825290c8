"""Timed cases of the token-model operators: layer norm and token embedding, each with its gradient.

Every case is one call of one operator on inputs a program has in hand.  `run` computes it in plain torch arithmetic
(32 bits, one rounding at the end), or, where `own` is true, through `hfuse_amd.ops`; `exact` evaluates the definition
in 64 bits.  All of them stream: `work` counts each input read once and each output written once.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-5


# ------------------------------------------------------------------------------------------------ cases
def _embed(op, tokens, vocab, cols, type, index="i64", spread="zipf", pad=False, out=None, **kw):
    return dict(kw, op=op, tokens=tokens, vocab=vocab, cols=cols, type=type, index=index, spread=spread, pad=pad,
                out=out or type)


def _norm(op, rows, cols, type, params=None, **kw):
    return dict(kw, op=op, rows=rows, cols=cols, type=type, params=params or type)


def listed():
    return [
        # one token of one sequence being generated: latency is all there is
        _embed("embedding", 1, 32000, 4096, "bf16", name="lookup-one"),
        # a ragged batch: row length and vocabulary odd, rows of half precision off every vector boundary, -1 behind the ends
        _embed("embedding", 4999, 32003, 1001, "f16", index="i32", spread="ragged", name="lookup-ragged"),
        # a training batch of 64 sequences of 2048 tokens
        _embed("embedding", 131072, 128000, 4096, "bf16", name="lookup-batch"),
        # fine-tuning on a few short lines in single precision: the gradient is nearly all zeros, and all of it is written
        _embed("embedding_backward", 256, 32000, 768, "f32", pad=True, name="table-grad-small"),
        # one micro-batch, gradient accumulated in single precision, ids uniform as after hashing
        _embed("embedding_backward", 16384, 50000, 2048, "bf16", spread="uniform", out="f32", name="table-grad-hashed"),
        # the training batch's gradient: few ids take most of the rows
        _embed("embedding_backward", 131072, 128000, 4096, "bf16", pad=True, name="table-grad-batch"),
        # the hidden state of one token being generated
        _norm("layer_norm", 1, 4096, "bf16", name="norm-one"),
        # odd rows in single precision
        _norm("layer_norm", 3001, 1155, "f32", name="norm-odd"),
        # a training batch of 32768 tokens at a wide model, parameters kept in single precision
        _norm("layer_norm", 32768, 8192, "bf16", params="f32", name="norm-batch"),
        # a short batch of a small model
        _norm("layer_norm_backward", 64, 1024, "bf16", params="f32", name="norm-grad-small"),
        # odd rows of half precision, none on a vector boundary
        _norm("layer_norm_backward", 5003, 1155, "f16", name="norm-grad-odd"),
        # the training batch again
        _norm("layer_norm_backward", 32768, 8192, "bf16", name="norm-grad-batch"),
    ]


def _spread(rng, lo, hi):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.4 and v >= 128:   # a good part of real sizes are multiples of 64
        v -= v % 64
    return max(lo, min(hi, v))


def draw(rng):
    type = rng.choice(("f32", "bf16", "bf16", "f16"))
    s = SIZES[type]
    cols = _spread(rng, 64, 8192)
    op = rng.choice(("embedding", "embedding_backward", "layer_norm", "layer_norm_backward"))
    if op.startswith("layer"):
        rows = _spread(rng, 1, 32768 * 2 // s)
        return _norm(op, rows, cols, type, params=rng.choice((type, "f32")))
    vocab = _spread(rng, 1000, 128000)
    tokens = _spread(rng, 1, 131072)
    if cols * s > 4096 * 2:   # no dearer than the largest listed
        vocab = max(1000, vocab * 8192 // (cols * s))
        tokens = max(1, tokens * 8192 // (cols * s))
    out = rng.choice((type, type, "f32")) if op == "embedding_backward" and cols * 4 <= 8192 else type
    return _embed(op, tokens, vocab, cols, type, index=rng.choice(("i64", "i32")),
                  spread=rng.choice(("zipf", "uniform", "ragged")), pad=rng.random() < 0.5, out=out)


# ------------------------------------------------------------------------------------------------ inputs
def _ids(case, g):
    """Token ids: log-uniform (the k-th most frequent with a probability of about 1 / k, low ids first, as a learnt
    vocabulary numbers them), uniform, or log-uniform with a sequence's unused end at -1."""
    n, v = case["tokens"], case["vocab"]
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    if case["spread"] == "uniform":
        t = (u * v).long()
    else:
        t = (torch.exp(u * math.log(v + 1.0)) - 1.0).long()
    t = t.clamp_(0, v - 1)
    if case["spread"] == "ragged":
        length = max(1, min(512, n // 4))
        used = torch.randint(1, length + 1, ((n + length - 1) // length,), generator=g, device="cuda")
        at = torch.arange(n, device="cuda")
        t = torch.where(at % length < used[at // length], t, torch.full_like(t, -1))
    return t.to(torch.int64 if case["index"] == "i64" else torch.int32)


def _hidden(rows, cols, type, g):
    """Hidden states: rows of different scale, an offset, and a few channels far larger than the rest."""
    x = torch.randn((rows, cols), generator=g, device="cuda")
    x *= 0.5 + torch.rand((rows, 1), generator=g, device="cuda")
    channel = torch.rand((cols,), generator=g, device="cuda")
    x *= torch.where(channel < 0.002, 20.0, 1.0)
    x += 0.3 * torch.randn((cols,), generator=g, device="cuda")
    return x.to(TYPES[type])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, type = case["op"], TYPES[case["type"]]
    state = {"case": case}
    if op.startswith("embedding"):
        state["tokens"] = _ids(case, g)
        state["scale"] = math.sqrt(case["cols"])
        if op == "embedding":
            state["weight"] = (0.02 * torch.randn((case["vocab"], case["cols"]), generator=g, device="cuda")).to(type)
        else:
            state["dy"] = (0.05 * torch.randn((case["tokens"], case["cols"]), generator=g, device="cuda")).to(type)
        return state
    rows, cols = case["rows"], case["cols"]
    x = state["x"] = _hidden(rows, cols, case["type"], g)
    params = TYPES[case["params"]]
    state["weight"] = (1.0 + 0.1 * torch.randn((cols,), generator=g, device="cuda")).to(params)
    state["bias"] = (0.1 * torch.randn((cols,), generator=g, device="cuda")).to(params)
    if op == "layer_norm_backward":
        state["dy"] = (0.05 * torch.randn((rows, cols), generator=g, device="cuda")).to(type)
        x32 = x.float()   # what the forward pass handed on
        mean = x32.mean(1, keepdim=True)
        state["mean"] = mean
        state["rstd"] = 1.0 / torch.sqrt(((x32 - mean) ** 2).mean(1, keepdim=True) + EPS)
    return state


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    return (_own if own else _plain)[case["op"]](state, case)


def _plain_embedding(s, case):
    t, w = s["tokens"].long(), s["weight"]
    used = (t >= 0) & (t < w.shape[0])
    rows = w[torch.where(used, t, torch.zeros_like(t))].float() * s["scale"]
    return torch.where(used[:, None], rows, torch.zeros_like(rows)).to(w.dtype)


def _plain_embedding_backward(s, case):
    t, dy = s["tokens"].long(), s["dy"]
    used = (t >= 0) & (t < case["vocab"])
    if case["pad"]:
        used &= t != 0
    dw = torch.zeros((case["vocab"], case["cols"]), device=dy.device)
    rows = torch.where(used[:, None], dy.float(), torch.zeros((), device=dy.device))
    dw.index_add_(0, torch.where(used, t, torch.zeros_like(t)), rows)
    return (dw * s["scale"]).to(TYPES[case["out"]])


def _plain_layer_norm(s, case):
    x = s["x"].float()
    mean = x.mean(1, keepdim=True)
    d = x - mean
    rstd = 1.0 / torch.sqrt((d * d).mean(1, keepdim=True) + EPS)
    y = d * rstd * s["weight"].float() + s["bias"].float()
    return y.to(s["x"].dtype), mean, rstd


def _plain_layer_norm_backward(s, case):
    dy, w = s["dy"].float(), s["weight"]
    h = (s["x"].float() - s["mean"]) * s["rstd"]
    g = dy * w.float()
    dx = s["rstd"] * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
    return dx.to(s["x"].dtype), (dy * h).sum(0).to(w.dtype), dy.sum(0).to(w.dtype)


def _own_embedding(s, case):
    from hfuse_amd import ops
    return ops.run(ops.embedding(s["tokens"], s["weight"], s["scale"]))[0]


def _own_embedding_backward(s, case):
    from hfuse_amd import ops
    return ops.run(ops.embedding_backward(s["dy"], s["tokens"], case["vocab"], s["scale"],
                                          padding_idx=0 if case["pad"] else None, dtype=TYPES[case["out"]]))[0]


def _own_layer_norm(s, case):
    from hfuse_amd import ops
    return ops.run(ops.layer_norm(s["x"], case["cols"], s["weight"], s["bias"], EPS))


def _own_layer_norm_backward(s, case):
    from hfuse_amd import ops
    return ops.run(ops.layer_norm_backward(s["dy"], s["x"], case["cols"], s["mean"], s["rstd"], s["weight"]))


_plain = {"embedding": _plain_embedding, "embedding_backward": _plain_embedding_backward,
          "layer_norm": _plain_layer_norm, "layer_norm_backward": _plain_layer_norm_backward}
_own = {"embedding": _own_embedding, "embedding_backward": _own_embedding_backward,
        "layer_norm": _own_layer_norm, "layer_norm_backward": _own_layer_norm_backward}


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "embedding":
        table = torch.cat([s["weight"].double() * s["scale"], s["weight"].new_zeros((1, case["cols"])).double()])
        return table.index_select(0, s["tokens"].long() % (case["vocab"] + 1))   # -1 is the row of zeros behind the table
    if op == "embedding_backward":
        t = s["tokens"].long()
        keep = torch.nonzero((t >= 0) & (t != (0 if case["pad"] else -1)))[:, 0]
        order = keep[torch.argsort(t[keep], stable=True)]
        ids, counts = torch.unique_consecutive(t[order], return_counts=True)
        out = torch.zeros((case["vocab"], case["cols"]), dtype=torch.float64, device="cuda")
        width = max(1, (1 << 28) // max(1, order.numel()))
        for c in range(0, case["cols"], width):   # running sums down the sorted rows, their differences at the ids' ends
            total = torch.cumsum(s["dy"][:, c:c + width].double()[order], 0)
            ends = total[torch.cumsum(counts, 0) - 1]
            out[ids, c:c + width] = torch.diff(ends, dim=0, prepend=torch.zeros_like(ends[:1])) * s["scale"]
        return out
    x = s["x"].double()
    n = case["cols"]
    if op == "layer_norm":
        mean = torch.sum(x, 1, keepdim=True) / n
        var = torch.sum(torch.square(x - mean), 1, keepdim=True) / n
        rstd = torch.rsqrt(var + EPS)
        return torch.addcmul(s["bias"].double(), (x - mean) * rstd, s["weight"].double()), mean, rstd
    rstd = s["rstd"].double()
    h = x.sub_(s["mean"].double()).mul_(rstd)
    dy = s["dy"].double()
    db, dw = torch.sum(dy, 0), torch.sum(dy * h, 0)
    g = dy.mul_(s["weight"].double())
    a = torch.sum(g, 1, keepdim=True) / n
    b = torch.sum(g * h, 1, keepdim=True) / n
    return g.sub_(a).sub_(h.mul_(b)).mul_(rstd), dw, db


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def _distinct(case):
    """Expected number of different ids in the batch."""
    n, v = case["tokens"], case["vocab"]
    if case["spread"] == "uniform":
        return v * -math.expm1(n * math.log1p(-1.0 / v))
    if case["spread"] == "ragged":
        n = (n + 1) // 2
    k = np.arange(1, v + 1, dtype=np.float64)
    return float(-np.expm1(n * np.log1p(-np.minimum(np.log((k + 1) / k) / math.log(v + 1.0), 1.0 - 1e-12))).sum())


def work(case):
    s, cols = SIZES[case["type"]], case["cols"]
    if case["op"].startswith("embedding"):
        n, ids = case["tokens"], case["tokens"] * (8 if case["index"] == "i64" else 4)
        if case["op"] == "embedding":
            return {"bytes": int(ids + _distinct(case) * cols * s + n * cols * s), "flops": n * cols}
        used = (n + 1) // 2 if case["spread"] == "ragged" else n
        return {"bytes": int(ids + used * cols * s + case["vocab"] * cols * SIZES[case["out"]]), "flops": used * cols}
    p, rows = SIZES[case["params"]], case["rows"]
    if case["op"] == "layer_norm":
        return {"bytes": 2 * rows * cols * s + 8 * rows + 2 * cols * p, "flops": 8 * rows * cols}
    return {"bytes": 3 * rows * cols * s + 8 * rows + 3 * cols * p, "flops": 14 * rows * cols}

"""The operators at the two ends and in the middle of an encoder-decoder language model, as cases that can be timed and compared: embedding rows of tokens, attention of
a decoder's positions to an encoder's states, and the cross entropy of a projection onto a large vocabulary whose logits are not kept; each with its gradient.

``run(state)`` makes one pass through one operator. With ``own`` set it is the call that a program makes of ``dali_amd.op``, into destinations that the program keeps;
otherwise the same formulas as elementary torch operations on the same values.
"""
import math

import torch

own = False

_TORCH = {"f32": torch.float32, "f64": torch.float64, "i32": torch.int32}
_SIZE = {"f32": 4, "f64": 8}


def listed():
    return [
        # A decoder's step: the embeddings of eight sequences' last tokens. Nothing but latency counts.
        {"name": "embed_8x1024", "kind": "embed", "tokens": 8, "rows": 32000, "width": 1024, "dtype": "f32"},
        # The tokens of a training batch of 256 sequences of 256 tokens, some of them padding ...
        {"name": "embed_65536x1024", "kind": "embed", "tokens": 65536, "rows": 32000, "width": 1024, "dtype": "f32"},
        # ... and the way back: as in texts, a few words make up much of the batch and most words are not in it.
        {"name": "embed_backward_65536x1024", "kind": "embed_backward", "tokens": 65536, "rows": 32000, "width": 1024, "dtype": "f32"},
        # A character set in double precision with odd sizes: every row is met by many tokens.
        {"name": "embed_backward_f64_3001x515", "kind": "embed_backward", "tokens": 3001, "rows": 97, "width": 515, "dtype": "f64"},
        # Answering: one position of each of 32 sequences looks at up to 2048 encoder states through four shared heads.
        {"name": "attention_32x1x2048", "kind": "attention", "batch": 32, "queries": 1, "keys": 2048, "heads": 16, "kv_heads": 4, "width": 64, "dtype": "f32"},
        # A training batch of a translation model ...
        {"name": "attention_16x256x512", "kind": "attention", "batch": 16, "queries": 256, "keys": 512, "heads": 16, "kv_heads": 16, "width": 64, "dtype": "f32"},
        # ... and the way back.
        {"name": "attention_backward_16x256x512", "kind": "attention_backward", "batch": 16, "queries": 256, "keys": 512, "heads": 16, "kv_heads": 16, "width": 64,
         "dtype": "f32"},
        # Long documents of odd lengths, wide heads, each shared by four.
        {"name": "attention_backward_2x1999x4001", "kind": "attention_backward", "batch": 2, "queries": 1999, "keys": 4001, "heads": 8, "kv_heads": 2, "width": 128,
         "dtype": "f32"},
        # Scoring the next token of eight sequences over a large vocabulary of odd size.
        {"name": "entropy_8x1024x50257", "kind": "entropy", "rows": 8, "inputs": 1024, "vocab": 50257, "dtype": "f32"},
        # The loss of a training batch of 32 sequences of 256 tokens ...
        {"name": "entropy_8192x1024x32000", "kind": "entropy", "rows": 8192, "inputs": 1024, "vocab": 32000, "dtype": "f32"},
        # ... and its gradients.
        {"name": "entropy_backward_8192x1024x32000", "kind": "entropy_backward", "rows": 8192, "inputs": 1024, "vocab": 32000, "dtype": "f32"},
        # Double precision with odd sizes: what a gradient check or a small exact model runs.
        {"name": "entropy_backward_f64_301x515x10007", "kind": "entropy_backward", "rows": 301, "inputs": 515, "vocab": 10007, "dtype": "f64"},
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], even over its logarithm; a third of them on the round numbers that programs like."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 1 / 3:
        v = next((v // step * step for step in (64, 16, 8) if v >= 2 * step), v)
    return max(low, min(high, v))


def draw(rng):
    kind = rng.choice(["embed", "embed_backward", "attention", "attention_backward", "entropy", "entropy_backward"])
    case = {"kind": kind}
    while True:
        case["dtype"] = rng.choice(["f32", "f32", "f32", "f64"])
        scores = 0
        if kind.startswith("embed"):
            case.update(tokens=_spread(rng, 1, 131072), rows=_spread(rng, 30, 131072), width=_spread(rng, 8, 4096))
        elif kind.startswith("attention"):
            kv_heads = rng.choice([1, 2, 4, 8, 16])
            case.update(batch=_spread(rng, 1, 64), queries=_spread(rng, 1, 2048), keys=_spread(rng, 1, 8192), heads=kv_heads * rng.choice([1, 1, 2, 4, 5]), kv_heads=kv_heads,
                        width=rng.choice([64, 128, 32, 256, _spread(rng, 16, 256)]))
            scores = case["batch"] * case["heads"] * case["queries"] * case["keys"]
        else:
            case.update(rows=_spread(rng, 1, 16384), inputs=_spread(rng, 16, 4096), vocab=_spread(rng, 30, 131072))
            scores = case["rows"] * case["vocab"]
        w = work(case)
        if w["bytes"] <= 8e8 and w["flops"] <= (1.2e12 if case["dtype"] == "f32" else 1e11) and scores <= (1 << 28):
            return case


# ------------------------------------------------------------------------------------------------ what a program has in hand
_TYPESTR = {"f32": "<f4", "f64": "<f8", "i32": "<i4"}


class _View(object):
    """Device memory of an array of the package for torch: no copy, and the array lives as long as the tensor."""

    def __init__(self, array, shape, dtype):
        self.array = array
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": _TYPESTR[dtype], "data": (array.device_ptr(), False), "version": 2}


class _Memory(object):
    """Tensors to fill, each in an array of the package where its operators are going to take it (they work on arrays of the package)."""

    def __init__(self):
        self.arrays = {}

    def __call__(self, name, shape, dtype):
        if not own:
            return torch.empty(shape, dtype=_TORCH[dtype], device="cuda")
        import dali_amd as D
        codes = {"f32": D.DTYPE_FLOAT, "f64": D.DTYPE_DOUBLE, "i32": D.DTYPE_INT32}
        array = self.arrays[name] = D.Array.empty(shape, codes[dtype])
        return torch.as_tensor(_View(array, shape, dtype), device="cuda")


def _counts(case):
    """How many of an encoder's states each sequence of a batch has: from half of the most to all of them, evenly."""
    batch, keys = case["batch"], case["keys"]
    return [keys - (keys // 2) * b // batch for b in range(batch)]


def _words(gen, n, rows):
    """Tokens as texts have them: the r-th most frequent one about 1 / r as often as the first, in no order of their numbers; one in twenty is padding (-1)."""
    u = torch.rand(n, device="cuda", dtype=torch.float64, generator=gen)
    rank = (torch.exp(u * math.log(rows + 1.0)) - 1.0).long().clamp_(0, rows - 1)
    tokens = torch.randperm(rows, device="cuda", generator=gen)[rank].int()
    padding = torch.rand(n, device="cuda", generator=gen) < 0.05
    return tokens.masked_fill_(padding, -1)


def prepare(case, seed):
    torch.cuda.synchronize()
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, dtype = case["kind"], case["dtype"]
    held, memory = {}, _Memory()

    def make(name, shape, type_=dtype):
        held[name] = memory(name, shape, type_)
        return held[name]

    def normal(name, shape, mean=0.0, scale=1.0):
        return make(name, shape).normal_(mean, scale, generator=gen)

    if kind.startswith("embed"):
        n, rows, width = case["tokens"], case["rows"], case["width"]
        make("tokens", (n,), "i32").copy_(_words(gen, n, rows))
        held["scale"] = math.sqrt(width)
        if kind == "embed":
            normal("table", (rows, width), 0.0, 1 / math.sqrt(width))
            outs = [make("y", (n, width))]
        else:
            normal("dy", (n, width))
            outs = [make("dtable", (rows, width))]
    elif kind.startswith("attention"):
        q_shape = (case["batch"], case["queries"], case["heads"], case["width"])
        k_shape = (case["batch"], case["keys"], case["kv_heads"], case["width"])
        normal("q", q_shape), normal("k", k_shape), normal("v", k_shape)
        order = torch.randperm(case["batch"], device="cuda", generator=gen)
        make("counts", (case["batch"],), "i32").copy_(torch.tensor(_counts(case), device="cuda")[order])
        held["scale"] = 1 / math.sqrt(case["width"])
        if kind == "attention":
            outs = [make("y", q_shape), make("lse", q_shape[:3])]
        else:
            normal("dy", q_shape)
            y, lse = _attention(held["q"], held["k"], held["v"], held["counts"], held["scale"])
            make("y", q_shape).copy_(y)
            make("lse", q_shape[:3]).copy_(lse)
            outs = [make("dq", q_shape), make("dk", k_shape), make("dv", k_shape)]
    else:
        rows, inputs, vocab = case["rows"], case["inputs"], case["vocab"]
        normal("x", (rows, inputs)), normal("w", (inputs, vocab), 0.0, 1.5 / math.sqrt(inputs)), normal("bias", (vocab,), 0.0, 0.2)
        make("targets", (rows,), "i32").copy_(_words(gen, rows, vocab))
        if kind == "entropy":
            outs = [make("losses", (rows,)), make("lse", (rows,))]
        else:
            _, lse = _entropy(held["x"], held["w"], held["bias"], held["targets"])
            make("lse", (rows,)).copy_(lse)
            make("d_losses", (rows,)).uniform_(0.5 / rows, 1.5 / rows, generator=gen)
            outs = [make("dx", (rows, inputs)), make("dw", (inputs, vocab)), make("dbias", (vocab,))]
    torch.cuda.synchronize()  # (the package works on a stream of its own)
    return {"case": dict(case), "held": held, "arrays": memory.arrays, "outs": outs}


# ------------------------------------------------------------------------------------------------ the plain forms
def _embed(table, tokens, scale):
    rows = table[tokens.clamp(min=0).long()] * scale
    return rows * (tokens >= 0)[:, None]


def _embed_backward(dy, tokens, rows, scale):
    given = torch.where((tokens >= 0)[:, None], dy, 0.0) * scale
    return torch.zeros((rows, dy.shape[1]), dtype=dy.dtype, device=dy.device).index_add_(0, tokens.clamp(min=0).long(), given)


def _by_kv_head(q, kv_heads):
    """[batch, kv_heads, the heads that share one and the positions, width]"""
    batch, queries, heads, width = q.shape
    return q.reshape(batch, queries, kv_heads, heads // kv_heads, width).permute(0, 2, 3, 1, 4).reshape(batch, kv_heads, heads // kv_heads * queries, width).contiguous()


def _by_position(rows, queries):
    """The way back: [batch, queries, heads, ...]"""
    batch, kv_heads, n = rows.shape[:3]
    split = rows.reshape((batch, kv_heads, n // queries, queries) + rows.shape[3:])
    return split.transpose(2, 3).transpose(1, 2).reshape((batch, queries, kv_heads * (n // queries)) + rows.shape[3:])


def _scores(q, k, counts, scale):
    q = _by_kv_head(q, k.shape[2])
    s = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()) * scale
    masked = torch.arange(k.shape[1], device=k.device)[None, :] >= counts[:, None]
    return q, s.masked_fill_(masked[:, None, None, :], -math.inf)


def _attention(q, k, v, counts, scale):
    _, s = _scores(q, k, counts, scale)
    top = s.max(3).values
    weight = torch.exp(s - top[..., None])
    total = weight.sum(3)
    y = torch.matmul(weight, v.permute(0, 2, 1, 3).contiguous()) / total[..., None]
    return _by_position(y, q.shape[1]), _by_position(top + torch.log(total), q.shape[1])


def _attention_backward(dy, q, k, v, y, lse, counts, scale):
    rows, s = _scores(q, k, counts, scale)
    kv_heads = k.shape[2]
    p = torch.exp(s - _by_kv_head(lse[..., None], kv_heads))
    dy_rows = _by_kv_head(dy, kv_heads)
    delta = (dy_rows * _by_kv_head(y, kv_heads)).sum(3)
    ds = p * (torch.matmul(dy_rows, v.permute(0, 2, 3, 1).contiguous()) - delta[..., None]) * scale
    dq = torch.matmul(ds, k.permute(0, 2, 1, 3).contiguous())
    dk = torch.matmul(ds.transpose(2, 3).contiguous(), rows)
    dv = torch.matmul(p.transpose(2, 3).contiguous(), dy_rows)
    return _by_position(dq, q.shape[1]), dk.transpose(1, 2).contiguous(), dv.transpose(1, 2).contiguous()


def _entropy(x, w, bias, targets):
    logits = torch.matmul(x, w) + bias
    top = logits.max(1).values
    log_total = torch.log(torch.exp(logits - top[:, None]).sum(1))
    chosen = logits.gather(1, targets.clamp(min=0).long()[:, None])[:, 0]
    return torch.where(targets >= 0, (top - chosen) + log_total, 0.0), top + log_total


def _entropy_backward(d_losses, x, w, bias, targets, lse):
    given = torch.where(targets >= 0, d_losses, 0.0)
    g = torch.exp(torch.matmul(x, w) + bias - lse[:, None]) * given[:, None]
    g.scatter_add_(1, targets.clamp(min=0).long()[:, None], -given[:, None])
    return torch.matmul(g, w.t()), torch.matmul(x.t(), g), g.sum(0)


def _plain(case, t):
    kind = case["kind"]
    if kind == "embed":
        return [_embed(t["table"], t["tokens"], t["scale"])]
    if kind == "embed_backward":
        return [_embed_backward(t["dy"], t["tokens"], case["rows"], t["scale"])]
    if kind == "attention":
        return list(_attention(t["q"], t["k"], t["v"], t["counts"], t["scale"]))
    if kind == "attention_backward":
        return list(_attention_backward(t["dy"], t["q"], t["k"], t["v"], t["y"], t["lse"], t["counts"], t["scale"]))
    if kind == "entropy":
        return list(_entropy(t["x"], t["w"], t["bias"], t["targets"]))
    return list(_entropy_backward(t["d_losses"], t["x"], t["w"], t["bias"], t["targets"], t["lse"]))


# ------------------------------------------------------------------------------------------------ the package's calls
def _own(case, t, a):
    from dali_amd import op
    kind = case["kind"]
    if kind == "embed":
        op.embedding(a["table"], a["tokens"], t["scale"], out=a["y"])
    elif kind == "embed_backward":
        op.embedding_backward(a["dy"], a["tokens"], case["rows"], t["scale"], out=a["dtable"])
    elif kind == "attention":
        op.cross_attention(a["q"], a["k"], a["v"], a["counts"], t["scale"], out=(a["y"], a["lse"]))
    elif kind == "attention_backward":
        op.cross_attention_backward(a["dy"], a["q"], a["k"], a["v"], a["y"], a["lse"], a["counts"], t["scale"], out=(a["dq"], a["dk"], a["dv"]))
    elif kind == "entropy":
        op.projected_cross_entropy(a["x"], a["w"], a["targets"], a["bias"], out=(a["losses"], a["lse"]))
    else:
        op.projected_cross_entropy_backward(a["d_losses"], a["x"], a["w"], a["targets"], a["lse"], a["bias"], out=(a["dx"], a["dw"], a["dbias"]))


def run(state):
    case = state["case"]
    if not own:
        return _plain(case, state["held"])
    _own(case, state["held"], state["arrays"])
    return state["outs"]


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def _exact_attention(case, t):
    """One sequence and one shared head after the other, over the states that there are."""
    outs = [torch.zeros_like(t["q"]), torch.zeros(t["q"].shape[:3], dtype=torch.float64, device="cuda")]
    if case["kind"] == "attention_backward":
        outs = [torch.zeros_like(t["q"]), torch.zeros_like(t["k"]), torch.zeros_like(t["v"])]
    group = case["heads"] // case["kv_heads"]
    for b, n in enumerate(t["counts"].tolist()):
        for h in range(case["heads"]):
            q, k, v = t["q"][b, :, h], t["k"][b, :n, h // group], t["v"][b, :n, h // group]
            s = (q @ k.t()) * t["scale"]
            if case["kind"] == "attention":
                outs[0][b, :, h] = torch.softmax(s, 1) @ v
                outs[1][b, :, h] = torch.logsumexp(s, 1)
                continue
            dy = t["dy"][b, :, h]
            p = torch.exp(s - t["lse"][b, :, h, None])
            ds = p * (dy @ v.t() - torch.einsum("td,td->t", dy, t["y"][b, :, h])[:, None])
            outs[0][b, :, h] = (ds @ k) * t["scale"]
            outs[1][b, :n, h // group] += (ds.t() @ q) * t["scale"]
            outs[2][b, :n, h // group] += p.t() @ dy
    return outs


def exact(case, seed):
    t = {k: v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for k, v in prepare(case, seed)["held"].items()}
    kind = case["kind"]
    if kind == "embed":
        with_padding = torch.cat([t["table"] * t["scale"], torch.zeros((1, case["width"]), dtype=torch.float64, device="cuda")])
        return [with_padding.index_select(0, torch.where(t["tokens"] < 0, case["rows"], t["tokens"]).long())]
    if kind == "embed_backward":
        # (row `rows` takes what padding has; as sums of runs of the tokens in their order)
        order = torch.sort(torch.where(t["tokens"] < 0, case["rows"], t["tokens"]).long(), stable=True)
        met, lengths = torch.unique_consecutive(order.values, return_counts=True)
        sums = torch.segment_reduce(t["dy"][order.indices], "sum", lengths=lengths, axis=0, unsafe=True) * t["scale"]
        out = torch.zeros((case["rows"] + 1, case["width"]), dtype=torch.float64, device="cuda")
        out[met] = sums
        return [out[:-1]]
    if kind.startswith("attention"):
        return _exact_attention(case, t)
    logits = torch.addmm(t["bias"], t["x"], t["w"])
    rows = torch.arange(case["rows"], device="cuda")
    there = t["targets"] >= 0
    chosen = torch.where(there, t["targets"], 0).long()
    if kind == "entropy":
        lse = torch.logsumexp(logits, 1)
        return [(lse - logits[rows, chosen]) * there, lse]
    g = logits.sub_(t["lse"][:, None]).exp_()
    g[rows, chosen] -= 1.0
    g *= (t["d_losses"] * there)[:, None]
    return [torch.mm(t["w"], g.t()).t(), torch.mm(g.t(), t["x"]).t(), torch.mv(g.t(), torch.ones(case["rows"], dtype=torch.float64, device="cuda"))]


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    kind, size = case["kind"], _SIZE[case["dtype"]]
    if kind.startswith("embed"):
        n, rows, width = case["tokens"], case["rows"], case["width"]
        # (tokens that come up again are read again from a cache: at least one row is read, and no more than there are)
        table = min(n, rows) if kind == "embed" else rows
        return {"bytes": size * width * (n + table) + 4 * n, "flops": n * width * (1 if kind == "embed" else 2)}
    if kind.startswith("attention"):
        q = case["batch"] * case["queries"] * case["heads"]
        states = sum(_counts(case))
        kv, pairs = states * case["kv_heads"] * case["width"], states * case["queries"] * case["heads"]
        if kind == "attention":
            return {"bytes": size * (2 * q * case["width"] + q + 2 * kv) + 4 * case["batch"], "flops": pairs * (4 * case["width"] + 4)}
        padded = case["batch"] * case["keys"] * case["kv_heads"] * case["width"]
        return {"bytes": size * (4 * q * case["width"] + q + 2 * kv + 2 * padded) + 4 * case["batch"], "flops": pairs * (10 * case["width"] + 6)}
    rows, inputs, vocab = case["rows"], case["inputs"], case["vocab"]
    weights = inputs * vocab + vocab
    if kind == "entropy":
        return {"bytes": size * (rows * inputs + weights + 2 * rows) + 4 * rows, "flops": rows * vocab * (2 * inputs + 4)}
    return {"bytes": size * (2 * rows * inputs + 2 * weights + 2 * rows) + 4 * rows, "flops": rows * vocab * (6 * inputs + 5)}

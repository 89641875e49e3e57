"""The operators that a language model is trained and scored with, as cases that can be timed and compared: layer normalisation, the log
probabilities of given tokens with entropy and top alternatives, each with its gradient, and clipping by the global norm of the gradients.

``run(state)`` makes one pass through one operator. With ``own`` set it is the call that a program makes of ``dali_amd.op``, into
destinations that the program keeps; otherwise the same formulas as elementary torch operations on the same values.
"""
import math
import random

import torch

own = False

_TORCH = {"f32": torch.float32, "f64": torch.float64, "i32": torch.int32}
_SIZE = {"f32": 4, "f64": 8}
EPSILON = 1e-5


def listed():
    return [
        # A decoder's step: the hidden states of eight sequences. Nothing but latency counts.
        {"name": "norm_8x1024", "kind": "norm", "rows": 8, "width": 1024, "dtype": "f32"},
        # The hidden states of a training batch of 32 sequences of 256 tokens ...
        {"name": "norm_8192x1024", "kind": "norm", "rows": 8192, "width": 1024, "dtype": "f32"},
        # ... and the way back.
        {"name": "norm_backward_8192x1024", "kind": "norm_backward", "rows": 8192, "width": 1024, "dtype": "f32"},
        # Double precision with odd sizes: what a gradient check or a small exact model runs.
        {"name": "norm_backward_f64_3001x2047", "kind": "norm_backward", "rows": 3001, "width": 2047, "dtype": "f64"},
        # The largest batch with wide rows.
        {"name": "norm_backward_32768x4096", "kind": "norm_backward", "rows": 32768, "width": 4096, "dtype": "f32"},
        # One answer, token by token: a single row of a large vocabulary of odd size, with twenty alternatives reported.
        {"name": "log_probs_1x50257", "kind": "log_probs", "rows": 1, "vocab": 50257, "alternatives": 20, "masked": False, "dtype": "f32"},
        # Eight sequences whose answers are constrained: half of the vocabulary is masked out.
        {"name": "log_probs_8x32000", "kind": "log_probs", "rows": 8, "vocab": 32000, "alternatives": 5, "masked": True, "dtype": "f32"},
        # Scoring a batch of texts.
        {"name": "log_probs_8192x32000", "kind": "log_probs", "rows": 8192, "vocab": 32000, "alternatives": 5, "masked": False, "dtype": "f32"},
        # The gradient of a training step's log probabilities and of an entropy bonus ...
        {"name": "log_probs_backward_8192x32000", "kind": "log_probs_backward", "rows": 8192, "vocab": 32000, "masked": False, "dtype": "f32"},
        # ... and over a character set: many positions, few and oddly many classes.
        {"name": "log_probs_backward_51200x97", "kind": "log_probs_backward", "rows": 51200, "vocab": 97, "masked": False, "dtype": "f32"},
        # The gradients of a character model: a dozen small tensors.
        {"name": "clip_12x40000", "kind": "clip", "tensors": 12, "largest": 40000, "spread": 3, "clipped": True, "dtype": "f32"},
        # The gradients of a two-layer model over 32000 words with 1024 hidden units: embedding, cells, norms, projection.
        {"name": "clip_24x33000000", "kind": "clip", "tensors": 24, "largest": 33000000, "spread": 7, "clipped": True, "dtype": "f32"},
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], even over its logarithm; a third of them on the round numbers that programs like."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 1 / 3:
        v = next((v // step * step for step in (64, 16, 8) if v >= 2 * step), v)
    return max(low, min(high, v))


def draw(rng):
    kind = rng.choice(["norm", "norm_backward", "log_probs", "log_probs_backward", "clip"])
    case = {"kind": kind}
    while True:
        case["dtype"] = rng.choice(["f32", "f32", "f32", "f64"])
        if kind in ("norm", "norm_backward"):
            case.update(rows=_spread(rng, 1, 65536), width=_spread(rng, 8, 16384))
        elif kind == "clip":
            case.update(tensors=_spread(rng, 1, 60), largest=_spread(rng, 100, 30000000), spread=rng.randrange(1000), clipped=rng.random() < 0.75)
        else:
            case.update(rows=_spread(rng, 1, 65536), vocab=_spread(rng, 30, 131072), masked=rng.random() < 0.25)
            if kind == "log_probs":
                case["alternatives"] = rng.choice([0, 1, 5, 5, 20])
        if work(case)["bytes"] <= 1.2e9:
            return case


def _shapes(case):
    """What the tensors of a model look like: matrices and the vectors beside them, the largest matrix first."""
    rng, largest = random.Random(case["spread"]), case["largest"]
    sizes = [largest] + [_spread(rng, max(1, largest // 200), largest // 4 + 1) for _ in range(case["tensors"] - 1)]
    columns = [max(1, math.isqrt(n) // 2) for n in sizes]
    return [(n // c, c) if i == 0 or rng.random() < 0.6 else (c,) for i, (n, c) in enumerate(zip(sizes, columns))]


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

    if kind in ("norm", "norm_backward"):
        rows, width = case["rows"], case["width"]
        x, gamma = normal("x", (rows, width), 0.3, 2.0), normal("gamma", (width,), 1.0, 0.2)
        if kind == "norm":
            normal("beta", (width,), 0.0, 0.2)
            outs = [make("y", (rows, width)), make("mean", (rows,)), make("rstd", (rows,))]
        else:
            normal("dy", (rows, width))
            _, mean, rstd = _norm(x, gamma, 0.0)
            make("mean", (rows,)).copy_(mean)
            make("rstd", (rows,)).copy_(rstd)
            outs = [make("dx", (rows, width)), make("dgamma", (width,)), make("dbeta", (width,))]
    elif kind == "clip":
        grads = [normal("grad%d" % i, s, 0.0, 0.01) for i, s in enumerate(_shapes(case))]
        norm = 0.01 * math.sqrt(sum(g.numel() for g in grads))
        held["max_norm"] = norm / 3 if case["clipped"] else norm * 3
        outs = [make("clipped%d" % i, g.shape) for i, g in enumerate(grads)] + [make("norm", ())]
    else:
        rows, vocab = case["rows"], case["vocab"]
        x = normal("logits", (rows, vocab), 0.0, 2.0)
        tokens = make("tokens", (rows,), "i32").random_(0, vocab, generator=gen)
        if case["masked"]:
            # half of the vocabulary is not to be said, in each row another half; the given token always may
            banned = torch.randint(0, 2, (rows, vocab), dtype=torch.uint8, device="cuda", generator=gen).bool()
            banned.scatter_(1, tokens.long()[:, None], False)
            x.masked_fill_(banned, -math.inf)
            del banned
        if kind == "log_probs":
            k = min(case["alternatives"], vocab)
            outs = [make("log_probs", (rows,)), make("entropy", (rows,)), make("lse", (rows,))]
            outs += [make("top_log_probs", (rows, k)), make("top_tokens", (rows, k), "i32")] if k else []
        else:
            _, entropy, lse = _log_probs(x, tokens)
            make("entropy", (rows,)).copy_(entropy)
            make("lse", (rows,)).copy_(lse)
            normal("d_log_probs", (rows,))
            normal("d_entropy", (rows,), 0.0, 0.1)
            outs = [make("d_logits", (rows, vocab))]
    torch.cuda.synchronize()  # (the package works on a stream of its own)
    return {"case": dict(case), "held": held, "arrays": memory.arrays, "outs": outs}


# ------------------------------------------------------------------------------------------------ the plain forms
def _norm(x, gamma, beta):
    mean = x.mean(1)
    centred = x - mean[:, None]
    rstd = 1.0 / torch.sqrt(centred.square().mean(1) + EPSILON)
    return centred * rstd[:, None] * gamma + beta, mean, rstd


def _norm_backward(dy, x, mean, rstd, gamma):
    normed = (x - mean[:, None]) * rstd[:, None]
    scaled = dy * gamma
    dx = rstd[:, None] * (scaled - scaled.mean(1)[:, None] - normed * (scaled * normed).mean(1)[:, None])
    return dx, (dy * normed).sum(0), dy.sum(0)


def _log_probs(x, tokens):
    top = x.max(1).values
    below = x - top[:, None]
    weight = torch.exp(below)
    total = weight.sum(1)
    # (a masked token adds nothing to the entropy)
    entropy = torch.log(total) - torch.where(weight > 0, weight * below, 0.0).sum(1) / total
    lse = top + torch.log(total)
    return x.gather(1, tokens.long()[:, None])[:, 0] - lse, entropy, lse


def _alternatives(x, k):
    """Positions of the k largest values of each row, the lower position first among equals."""
    if x.dtype == torch.float64:
        return torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k]
    bits = (x + 0.0).view(torch.int32)
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    positions = torch.arange(x.shape[1], device=x.device)
    return (x.shape[1] - 1 - torch.topk((order << 32) + (x.shape[1] - 1 - positions), k, dim=1).values.bitwise_and_(0xFFFFFFFF)).int()


def _log_probs_backward(g, h, x, tokens, lse, entropy):
    log_p = x - lse[:, None]
    p = torch.exp(log_p)
    dx = -p * g[:, None] - torch.where(p > 0, p * (log_p + entropy[:, None]), 0.0) * h[:, None]
    return dx.scatter_add_(1, tokens.long()[:, None], g[:, None])


def _plain(case, t):
    kind = case["kind"]
    if kind == "norm":
        return list(_norm(t["x"], t["gamma"], t["beta"]))
    if kind == "norm_backward":
        return list(_norm_backward(t["dy"], t["x"], t["mean"], t["rstd"], t["gamma"]))
    if kind == "log_probs":
        log_probs, entropy, lse = _log_probs(t["logits"], t["tokens"])
        k = min(case["alternatives"], case["vocab"])
        if not k:
            return [log_probs, entropy, lse]
        top = _alternatives(t["logits"], k)
        return [log_probs, entropy, lse, t["logits"].gather(1, top.long()) - lse[:, None], top.int()]
    if kind == "log_probs_backward":
        return [_log_probs_backward(t["d_log_probs"], t["d_entropy"], t["logits"], t["tokens"], t["lse"], t["entropy"])]
    grads = [t["grad%d" % i] for i in range(case["tensors"])]
    norm = torch.stack([g.square().sum() for g in grads]).sum().sqrt()
    scale = torch.where(norm > t["max_norm"], t["max_norm"] / norm, 1.0).to(norm.dtype)
    return [g * scale for g in grads] + [norm]


# ------------------------------------------------------------------------------------------------ the package's calls
def _own(case, t, a):
    from dali_amd import op
    kind = case["kind"]
    if kind == "norm":
        op.layer_norm(a["x"], a["gamma"], a["beta"], EPSILON, out=(a["y"], a["mean"], a["rstd"]))
    elif kind == "norm_backward":
        op.layer_norm_backward(a["dy"], a["x"], a["mean"], a["rstd"], a["gamma"], out=(a["dx"], a["dgamma"], a["dbeta"]))
    elif kind == "log_probs":
        k = min(case["alternatives"], case["vocab"])
        top = (a["top_log_probs"], a["top_tokens"]) if k else (None, None)
        op.token_log_probs(a["logits"], a["tokens"], k, out=(a["log_probs"], a["entropy"], a["lse"]) + top)
    elif kind == "log_probs_backward":
        op.token_log_probs_backward(a["d_log_probs"], a["d_entropy"], a["logits"], a["tokens"], a["lse"], a["entropy"], out=a["d_logits"])
    else:
        n = case["tensors"]
        op.clip_by_global_norm([a["grad%d" % i] for i in range(n)], t["max_norm"], out=([a["clipped%d" % i] for i in range(n)], a["norm"]))


def run(state):
    case = state["case"]
    if not own:
        return _plain(case, state["held"])
    _own(case, state["held"], state["arrays"])
    return state["outs"]


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    t = {k: v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for k, v in prepare(case, seed)["held"].items()}
    kind = case["kind"]
    if kind in ("norm", "norm_backward"):
        x, n = t["x"], case["width"]
        if kind == "norm":
            mean = x.sum(1) / n
            variance = (x - mean[:, None]).pow(2).sum(1) / n
            rstd = (variance + EPSILON).pow(-0.5)
            return [torch.addcmul(t["beta"], (x - mean[:, None]) / (variance + EPSILON).sqrt()[:, None], t["gamma"]), mean, rstd]
        unit = torch.addcmul((-t["mean"] * t["rstd"])[:, None], x, t["rstd"][:, None])
        a = t["dy"] * t["gamma"]
        along, level = (a * unit).sum(1) / n, a.sum(1) / n
        dx = (a - torch.addcmul(level[:, None], unit, along[:, None])) * t["rstd"][:, None]
        return [dx, unit.mul_(t["dy"]).sum(0), torch.ones(case["rows"], dtype=torch.float64, device=x.device) @ t["dy"]]
    if kind == "clip":
        grads = [t["grad%d" % i] for i in range(case["tensors"])]
        norm = math.sqrt(math.fsum(float(torch.dot(g.reshape(-1), g.reshape(-1))) for g in grads))
        return [g * min(1.0, t["max_norm"] / norm) for g in grads] + [torch.tensor(norm, dtype=torch.float64)]
    x, rows = t["logits"], torch.arange(case["rows"], device=t["logits"].device)
    if kind == "log_probs":
        lse = torch.logsumexp(x, 1)
        p = torch.exp(x - lse[:, None])
        entropy = lse - torch.nan_to_num(p * x, nan=0.0).sum(1)
        outs = [x[rows, t["tokens"].long()] - lse, entropy, lse]
        k = min(case["alternatives"], case["vocab"])
        if k:
            outs += [torch.topk(x, k, dim=1).values - lse[:, None], None]
        return outs
    p = torch.exp(x - t["lse"][:, None])
    surprise = torch.where(p > 0, t["lse"][:, None] - x, 0.0)
    dx = p * (t["d_entropy"][:, None] * (surprise - t["entropy"][:, None]) - t["d_log_probs"][:, None])
    dx[rows, t["tokens"].long()] += t["d_log_probs"]
    return [dx]


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    kind, size = case["kind"], _SIZE[case["dtype"]]
    if kind == "norm":
        n = case["rows"] * case["width"]
        return {"bytes": size * (2 * n + 2 * case["width"] + 2 * case["rows"]), "flops": 8 * n}
    if kind == "norm_backward":
        n = case["rows"] * case["width"]
        return {"bytes": size * (3 * n + 3 * case["width"] + 2 * case["rows"]), "flops": 14 * n}
    if kind == "clip":
        n = sum(math.prod(s) for s in _shapes(case))
        return {"bytes": size * (2 * n + 1), "flops": 3 * n}
    n, rows = case["rows"] * case["vocab"], case["rows"]
    if kind == "log_probs":
        k = min(case["alternatives"], case["vocab"])
        return {"bytes": size * (n + rows * (3 + k)) + 4 * rows * (1 + k), "flops": 6 * n}
    return {"bytes": size * (2 * n + 4 * rows) + 4 * rows, "flops": 9 * n}

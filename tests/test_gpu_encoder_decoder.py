"""The operators of an encoder-decoder model together, as a program uses them: a training step with a table that is shared by the embeddings of both sides and the projection, eager
and recorded, against automatic differentiation in 64 bits on the CPU; and a decoder's step, one position at a time, against the whole sequence at once."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


class Model(object):
    def __init__(self, rng, vocab, heads, kv_heads, width, dtype):
        self.vocab, self.heads, self.kv_heads, self.width, self.dtype = vocab, heads, kv_heads, width, dtype
        d = heads * width
        make = lambda *s: (rng.randn(*s) / np.sqrt(s[0])).astype(dtype)  # noqa: E731
        self.table = (rng.randn(vocab, d) / np.sqrt(d)).astype(dtype)
        self.wq, self.wk, self.wv, self.wo = make(d, d), make(d, kv_heads * width), make(d, kv_heads * width), make(d, d)
        self.bias = (0.1 * rng.randn(vocab)).astype(dtype)
        self.scale = float(np.sqrt(d))

    NAMES = ("table", "wq", "wk", "wv", "wo", "bias")


def by_torch(m, source, counts, given, follows):
    p = {n: torch.tensor(getattr(m, n).astype(np.float64), requires_grad=True) for n in m.NAMES}
    b, t = given.shape
    rows = lambda tokens: p["table"][torch.tensor(np.maximum(tokens, 0)).long()] * m.scale * torch.tensor(tokens >= 0)[..., None]  # noqa: E731
    e, x = rows(source), rows(given)
    group = m.heads // m.kv_heads
    q = (x @ p["wq"]).reshape(b, t, m.heads, m.width)
    k = (e @ p["wk"]).reshape(b, -1, m.kv_heads, m.width).repeat_interleave(group, 2)
    v = (e @ p["wv"]).reshape(b, -1, m.kv_heads, m.width).repeat_interleave(group, 2)
    s = torch.einsum("bthd,bshd->bhts", q, k) / m.width ** 0.5
    s = s.masked_fill(torch.arange(k.shape[1])[None, None, None, :] >= torch.tensor(counts)[:, None, None, None], -np.inf)
    y = torch.einsum("bhts,bshd->bthd", torch.softmax(s, -1), v).reshape(b, t, -1)
    h = y @ p["wo"] + x
    logits = h @ p["table"].t() + p["bias"]
    there = torch.tensor(follows >= 0)
    losses = -torch.log_softmax(logits, -1).gather(-1, torch.tensor(np.maximum(follows, 0)).long()[..., None])[..., 0] * there
    loss = losses.sum() / there.sum()
    loss.backward()
    return losses.detach().numpy(), [p[n].grad.numpy() for n in m.NAMES]


class Step(object):
    """A training step on arrays that stay, so that it can be recorded"""

    def __init__(self, D, m, source, counts, given, follows):
        A = D.Array.from_numpy
        self.D, self.m = D, m
        self.p = {n: A(getattr(m, n)) for n in m.NAMES}
        self.source, self.counts, self.given, self.follows = A(source), A(counts), A(given), A(follows)
        self.d_losses = A((np.ones(follows.shape) / (follows >= 0).sum()).astype(m.dtype))

    def run(self):
        op, m, p = self.D.op, self.m, self.p
        b, t = self.given.shape
        s, d, kv = self.source.shape[1], m.heads * m.width, m.kv_heads * m.width
        dot = lambda a, w: op.dot(a, w).eval()  # noqa: E731
        e = op.embedding(p["table"], self.source, m.scale).reshape(b * s, d)
        x = op.embedding(p["table"], self.given, m.scale).reshape(b * t, d)
        q, k, v = dot(x, p["wq"]).reshape(b, t, m.heads, m.width), dot(e, p["wk"]).reshape(b, s, m.kv_heads, m.width), dot(e, p["wv"]).reshape(b, s, m.kv_heads, m.width)
        y, lse = op.cross_attention(q, k, v, self.counts)
        flat = y.reshape(b * t, d)
        h = (dot(flat, p["wo"]) + x).eval()
        follows, d_losses = self.follows.reshape(b * t), self.d_losses.reshape(b * t)
        losses, level = op.projected_cross_entropy(h, p["table"].T, follows, p["bias"])
        dh, dw, dbias = op.projected_cross_entropy_backward(d_losses, h, p["table"].T, follows, level, p["bias"])
        dwo, dy = dot(flat.T, dh), dot(dh, p["wo"].T).reshape(b, t, m.heads, m.width)
        dq, dk, dv = op.cross_attention_backward(dy, q, k, v, y, lse, self.counts)
        dq, dk, dv = dq.reshape(b * t, d), dk.reshape(b * s, kv), dv.reshape(b * s, kv)
        dx = (dh + dot(dq, p["wq"].T)).eval()
        de = (dot(dk, p["wk"].T) + dot(dv, p["wv"].T)).eval()
        dtable = (dw.T + op.embedding_backward(dx.reshape(b, t, d), self.given, m.vocab, m.scale) + op.embedding_backward(de.reshape(b, s, d), self.source, m.vocab, m.scale)).eval()
        return losses, [dtable, dot(x.T, dq), dot(e.T, dk), dot(e.T, dv), dwo, dbias]


def batch(rng, vocab, b, s, t):
    counts = np.array([s - (s // 2) * i // b for i in range(b)], np.int32)
    source, given, follows = (rng.randint(0, vocab, (b, n)).astype(np.int32) for n in (s, t, t))
    source[np.arange(s)[None, :] >= counts[:, None]] = -1
    given[0, t // 2:], follows[0, t // 2:] = -1, -1
    return source, counts, given, follows


def near(got, want, inner, dtype):
    """Ten stages at most, each a sum over `inner` products: off by ten times inner u of the norm, if nothing cancels; a factor of 4 for what does (the softmax's gradients)."""
    bound = 4 * 10 * inner * np.finfo(dtype).eps / 2
    return np.linalg.norm(got - want) <= bound * np.linalg.norm(want)


CASES = [(np.float64, 61, 4, 2, 8, (3, 11, 7)), (np.float32, 61, 4, 2, 8, (3, 11, 7)), (np.float64, 500, 6, 6, 20, (2, 70, 50)), (np.float32, 500, 2, 1, 64, (4, 150, 130)),
         (np.float32, 9000, 2, 2, 32, (8, 90, 70))]  # (the last one's projection goes by images)


@pytest.mark.parametrize("dtype,vocab,heads,kv_heads,width,shape", CASES)
def test_a_training_step(gpu, D, rng, dtype, vocab, heads, kv_heads, width, shape):
    m = Model(rng, vocab, heads, kv_heads, width, dtype)
    data = batch(rng, vocab, *shape)
    inner = max(heads * width, vocab, shape[0] * max(shape[1:]))
    want_losses, want = by_torch(m, *data)
    step = Step(D, m, *data)
    losses, gradients = step.run()
    assert near(losses.numpy(), want_losses.reshape(-1), inner, dtype)
    for name, g, w in zip(m.NAMES, gradients, want):
        assert near(g.numpy(), w, inner, dtype), name
    # recorded, and replayed with other parameters between the replays
    rec = D.Recording()
    with rec:
        losses, gradients = step.run()
    rec.make_graph()
    for turn in range(3):
        for n in ("table", "wq"):
            moved = (getattr(m, n) * (1.0 - 0.1 * (turn + 1))).astype(dtype)
            setattr(m, n, moved)
            step.p[n].assign(D.Array.from_numpy(moved))
        want_losses, want = by_torch(m, *data)
        rec.replay()
        assert near(losses.numpy(), want_losses.reshape(-1), inner, dtype)
        for name, g, w in zip(m.NAMES, gradients, want):
            assert near(g.numpy(), w, inner, dtype), name
        eager, _ = step.run()  # the program's own work in between
        assert np.array_equal(eager.numpy(), losses.numpy())


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_a_decoders_steps(gpu, D, rng, dtype):
    """One position at a time, over keys and values that are made once."""
    A, op = D.Array.from_numpy, D.op
    m = Model(rng, 700, 8, 2, 32, dtype)
    source, counts, given, follows = batch(rng, 700, 5, 90, 6)
    d, kv = 256, 64
    e = op.embedding(A(m.table), A(source), m.scale).reshape(5 * 90, d)
    k, v = (op.dot(e, A(w)).eval().reshape(5, 90, 2, 32) for w in (m.wk, m.wv))
    want, _ = by_torch(m, source, counts, given, follows)
    for i in range(6):
        x = op.embedding(A(m.table), A(np.ascontiguousarray(given[:, i])), m.scale)
        y, _ = op.cross_attention(op.dot(x, A(m.wq)).eval().reshape(5, 1, 8, 32), k, v, A(counts))
        h = (op.dot(y.reshape(5, d), A(m.wo)) + x).eval()
        losses, _ = op.projected_cross_entropy(h, A(m.table).T, A(np.ascontiguousarray(follows[:, i])), A(m.bias))
        assert near(losses.numpy(), want[:, i], 700, dtype)

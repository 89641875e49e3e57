"""fp32 values that go to the bf16 matrix cores in three pieces: each kernel that cuts an operand, on operands that make the cut nearly all that its result can be off by. Bounds are in
the 2-norm and small enough that a kernel that lost a value's third piece would fail them, which every test shows by an oracle whose operand holds two.

u is half a unit in the last place of 1. A sum of n products goes through the matrix instruction sixteen at a time, six times (once for each product of pieces that is taken): each of these
6 ceil(n / 16) additions rounds a partial sum of about the result's size at most, which independent roundings bring to sqrt(6 ceil(n / 16)) u; the pieces that are left out, the end of
the chain and the last operation beside it are worth 4 u. Operands that are zero, or so few bits that their products are exact, add nothing.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def two(x):
    """What two bf16 pieces of fp32 values hold, in 64 bits"""
    def piece(v):
        bits = v.astype(np.float32).view(np.uint32).astype(np.uint64)
        return ((bits + 0x7fff + ((bits >> np.uint64(16)) & np.uint64(1))) & np.uint64(0xffff0000)).astype(np.uint32).view(np.float32).astype(np.float64)
    high = piece(x)
    return high + piece((x - high).astype(np.float32))


def chain(n):
    return np.sqrt(6.0 * -(-n // 16)) + 4.0


def norm(x):
    return np.sqrt((np.asarray(x, np.float64) ** 2).sum())


def check(got, want, bound, lost):
    """`bound` relative to the norm of `want`; `lost`: what operands of two pieces come to"""
    assert norm(got - want) <= bound * U * norm(want), norm(got - want) / norm(want) / U
    for one in lost:
        assert norm(one - want) > bound * U * norm(want), norm(one - want) / norm(want) / U


# ---------------------------------------------------------------------------------------------- attention
WIDTHS = [32, 64, 128, 256]
QUERIES = 70  # (more rows than the kernels of few rows take)


@pytest.mark.parametrize("width", WIDTHS)
def test_scores_and_values(gpu, D, rng, width):
    """One state: lse is the score, off by the factor of q (2 u), the chain and three roundings of lse; y is the value."""
    A = D.Array.from_numpy
    q, k, v = (rng.randn(5, n, 2, width).astype(np.float32) for n in (QUERIES, 1, 1))
    y, lse = (a.numpy() for a in D.op.cross_attention(A(q), A(k), A(v), None, 0.5))
    score = lambda a, b: (a.astype(np.float64) * b.astype(np.float64)).sum(-1) * 0.5  # noqa: E731
    check(lse, score(q, k), chain(width) + 5, [score(two(q), k), score(q, two(k))] if width < 128 else [score(two(q), two(k))])
    values = np.broadcast_to(v, q.shape)
    check(y, values, 4, [np.broadcast_to(two(v), q.shape)])


@pytest.mark.parametrize("width", WIDTHS)
def test_weights(gpu, D, rng, width):
    """Scores that are exact (a scale of ln 2, powers of two in q and few bits in k): weights of 1 and 2^-s. Only the second state has a value, 1: y is w / (1 + w)."""
    A = D.Array.from_numpy
    q, k, v = np.zeros((1, QUERIES, 1, width), np.float32), np.zeros((1, 2, 1, width), np.float32), np.zeros((1, 2, 1, width), np.float32)
    q[0, :, 0, 0] = -np.arange(1, QUERIES + 1) / 64.0
    k[0, 1, 0, 0], v[0, 1] = 1.0, 1.0
    y = D.op.cross_attention(A(q), A(k), A(v), None, np.log(2.0))[0].numpy()
    w = np.exp2(q[..., :1].astype(np.float64)) * np.ones(width)
    check(y, w / (1 + w), 2 + 6, [two(w.astype(np.float32)) / (1 + w)])


@pytest.mark.parametrize("width", WIDTHS)
def test_gradients_of_uniform_weights(gpu, D, rng, width):
    """All scores are 0, of two states: p = 1/2, off by 2 u. dv = sum p dy. With dy and v of few bits ds is exact: dq = scale sum ds k, dk = scale sum ds q (q and k in turn are 0)."""
    A, op, rows = D.Array.from_numpy, D.op, 32
    zero = lambda n: np.zeros((3, n, 1, width), np.float32)  # noqa: E731
    few = lambda n: rng.randint(-3, 4, (3, n, 1, width)).astype(np.float32)  # noqa: E731
    many = lambda n: rng.randn(3, n, 1, width).astype(np.float32)  # noqa: E731
    lse = np.full((3, rows, 1), np.log(2.0), np.float32)

    def gradients(q, k, v, dy, y):
        return [g.numpy() for g in op.cross_attention_backward(A(dy), A(q), A(k), A(v), A(y), A(lse), None, 0.5)]

    def exact(q, k, v, dy, y):
        q, k, v, dy, y = (a[:, :, 0].astype(np.float64) for a in (q, k, v, dy, y))
        ds = 0.5 * (np.matmul(dy, v.transpose(0, 2, 1)) - (dy * y).sum(-1, keepdims=True))
        dv = 0.5 * np.broadcast_to(dy.sum(1, keepdims=True), v.shape)
        return [a[:, :, None] for a in (0.5 * np.matmul(ds, k), 0.5 * np.matmul(ds.transpose(0, 2, 1), q), dv)]

    dy = many(rows)
    args = zero(rows), zero(2), zero(2), dy, zero(rows)
    check(gradients(*args)[2], exact(*args)[2], 2 + chain(rows), [exact(*args[:3], two(dy), args[4])[2]])
    v, dy = few(2), few(rows)
    y = np.broadcast_to(0.5 * (v[:, :1] + v[:, 1:]), (3, rows, 1, width)).astype(np.float32)
    q, k = many(rows), many(2)
    got, want = gradients(q, zero(2), v, dy, y), exact(q, zero(2), v, dy, y)
    check(got[1], want[1], 3 + chain(rows), [exact(two(q), zero(2), v, dy, y)[1]])
    got, want = gradients(zero(rows), k, v, dy, y), exact(zero(rows), k, v, dy, y)
    check(got[0], want[0], 3 + chain(2), [exact(zero(rows), two(k), v, dy, y)[0]])


@pytest.mark.parametrize("width", WIDTHS)
def test_gradients_of_weights(gpu, D, rng, width):
    """dy.v, with y given as 0 so that nothing is taken from it, and a single 1 in k: dq has ds in one place."""
    A, rows = D.Array.from_numpy, 64
    q, k, v, dy = np.zeros((3, rows, 1, width), np.float32), np.zeros((3, 2, 1, width), np.float32), rng.randn(3, 2, 1, width), rng.randn(3, rows, 1, width)
    v, dy = v.astype(np.float32), dy.astype(np.float32)
    k[:, 0, :, 0] = 1.0
    dq = D.op.cross_attention_backward(A(dy), A(q), A(k), A(v), A(q), A(np.full((3, rows, 1), np.log(2.0), np.float32)), None, 1.0)[0].numpy()
    ds = lambda a, b: 0.5 * (a.astype(np.float64) * b[:, :1].astype(np.float64)).sum(-1)  # noqa: E731
    assert (dq[..., 1:] == 0).all()
    check(dq[..., 0], ds(dy, v), 4 + chain(width), [ds(two(dy), two(v))])


@pytest.mark.parametrize("width", WIDTHS)
def test_gradients_of_scores(gpu, D, rng, width):
    """Scores of q and k on the way back: with an lse of 0, p = e^s, and the gradient of a value whose row has dy = 1 in one place is the sum of them. A score of about 2 is off by its
    factor and chain (of 32 values: the others of q are 0); exponents are rounded to multiples of 2^-20 beside the 16 that scales the pieces (8 u once, as the rows' level is 0), the
    exponential by 2 u."""
    A, rows = D.Array.from_numpy, 64
    q, k = rng.randn(3, rows, 1, width).astype(np.float32), rng.randn(3, 40, 1, width).astype(np.float32)
    q[..., :-32] = 0
    scale = 2.0 / np.sqrt(32)
    dy = np.zeros((3, rows, 1, width), np.float32)
    at = 17
    dy[:, at, :, 0] = 1.0
    dv = D.op.cross_attention_backward(A(dy), A(q), A(k), A(k), A(0 * q), A(np.zeros((3, rows, 1), np.float32)), None, scale)[2].numpy()
    p = lambda a, b: np.exp(np.matmul(b[:, :, 0].astype(np.float64), a[:, at, 0, :, None].astype(np.float64))[..., 0] * scale)  # noqa: E731
    want = p(q, k)
    # (relative to p: an error of the score, whose size is about 2 and up to ln of the largest p)
    size = np.log(want.max())
    check(dv[:, :, 0, 0], want, (chain(32) + 3) * size + 8 + 4, [p(two(q), two(k))])


# ---------------------------------------------------------------------------------------------- cross entropy of a projection
ROWS, INPUTS, VOCAB = 512, 16, 8192


def some_words(rng, size):
    """A vocabulary of which eight neighbours are not masked"""
    x, w, bias = rng.randn(ROWS, INPUTS).astype(np.float32), (rng.randn(INPUTS, VOCAB) * size / np.sqrt(INPUTS)).astype(np.float32), np.full(VOCAB, -np.inf, np.float32)
    words = np.arange(4096, 4104)
    bias[words] = 0
    return x, w, bias, words, rng.choice(words, ROWS).astype(np.int32)


def softmax(x, w, words):
    logits = x.astype(np.float64) @ w[:, words].astype(np.float64)
    top = logits.max(1, keepdims=True)
    lse = top + np.log(np.exp(logits - top).sum(1, keepdims=True))
    return logits, lse[:, 0], np.exp(logits - lse)


def test_logits(gpu, D, rng):
    """Losses of logits of about 30: off by the logits of the maximum and the target and three roundings."""
    A = D.Array.from_numpy
    x, w, bias, words, targets = some_words(rng, 30.0)

    def losses(x, w):
        logits, lse, _ = softmax(x, w, words)
        return lse - logits[np.arange(ROWS), targets - words[0]]

    want = losses(x, w)
    logits = softmax(x, w, words)[0]
    got = D.op.projected_cross_entropy(A(x), A(w), A(targets), A(bias))[0].numpy()
    bound = chain(INPUTS) * (norm(logits.max(1)) + norm(logits[np.arange(ROWS), targets - words[0]])) / norm(want) + 3
    check(got, want, bound, [losses(two(x), two(w))])


def test_gradient_of_the_rows(gpu, D, rng):
    """dx = g w^T over eight words whose p is about 1/8: p is off by 2 |l - lse| + 6 and the logit's error, g by 2 u."""
    A = D.Array.from_numpy
    x, w, bias, words, targets = some_words(rng, 0.2)
    d = rng.uniform(0.5, 1.5, ROWS).astype(np.float32)
    lse = softmax(x, w, words)[1].astype(np.float32)
    logits = softmax(x, w, words)[0]
    p = np.exp(logits - lse.astype(np.float64)[:, None])
    g = p.copy()
    g[np.arange(ROWS), targets - words[0]] -= 1
    g *= d[:, None].astype(np.float64)
    want = g @ w[:, words].astype(np.float64).T
    dx = D.op.projected_cross_entropy_backward(A(d), A(x), A(w), A(targets), A(lse), A(bias))[0].numpy()
    of_p = (2 * np.abs(logits - lse[:, None]).max() + 6 + chain(INPUTS) * np.abs(logits).max()) * norm(p * d[:, None]) / norm(g)
    check(dx, want, chain(8) + 2 + of_p, [g @ two(w[:, words]).T])
    assert norm(two(g.astype(np.float32)) @ w[:, words].astype(np.float64).T - want) > (chain(8) + 2 + of_p) * U * norm(want)


def test_gradient_of_the_weights(gpu, D, rng):
    """dw = x^T g of eight rows with targets of their own: the entries of the targets are nearly all of its norm, the other words' (whose p is off by 26 u and more) about 1/30."""
    A = D.Array.from_numpy
    x, w = rng.randn(ROWS, INPUTS).astype(np.float32), (rng.randn(INPUTS, VOCAB) * 1.5 / np.sqrt(INPUTS)).astype(np.float32)
    rows = np.arange(8) * 61 + 3
    targets, d = np.full(ROWS, -1, np.int32), rng.uniform(0.5, 1.5, ROWS).astype(np.float32)
    targets[rows] = rng.choice(VOCAB, 8, replace=False)
    logits = x.astype(np.float64) @ w.astype(np.float64)
    lse = np.log(np.exp(logits).sum(1)).astype(np.float32)
    p = np.exp(logits[rows] - lse[rows].astype(np.float64)[:, None])
    g = p.copy()
    g[np.arange(8), targets[rows]] -= 1
    g *= d[rows, None].astype(np.float64)
    want = x[rows].astype(np.float64).T @ g
    dw = D.op.projected_cross_entropy_backward(A(d), A(x), A(w), A(targets), A(lse))[1].numpy()
    of_p = (2 * np.abs(logits[rows] - lse[rows, None]).max() + 6 + chain(INPUTS) * np.abs(logits[rows]).max()) * norm(p * d[rows, None]) / norm(g)
    bound = chain(8 * 16) + 2 + of_p
    check(dw, want, bound, [two(x[rows]).T @ g, x[rows].astype(np.float64).T @ two(g.astype(np.float32))])

"""Log probabilities of tokens, entropy, alternatives and their gradient against the definition in higher precision: sizes around every change of the kernels, masks that
leave few entries or none, ties, infinities, views, destinations.

u is half a unit in the last place of 1. A weight e^d carries the rounding of d and of the exponential, (3 |d| + 4) u of it; a sum of n weights is at most n / 64
additions deep for one thread and some more over a workgroup.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = {np.float32: 2.0 ** -24, np.float64: 2.0 ** -53}
VOCABS = [1, 2, 3, 5, 31, 64, 65, 97, 128, 255, 256, 257, 500, 511, 512, 513, 1000, 1023, 1024, 1025, 2048, 2049, 3000, 4096, 4099, 8191, 8192, 16385, 32000, 50257, 70001]


def oracle(x, tokens):
    """lse, log probability, entropy and the bounds of their errors."""
    u = U[x.dtype.type]
    x = x.astype(np.longdouble)
    rows, n = x.shape
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        m = x.max(1)
        base = np.where(np.isneginf(m), 0, m)
        d = x - base[:, None]
        w = np.exp(d)
        s = w.sum(1)
        lse = base + np.log(s)
        p = np.where(w > 0, w, 0) / np.where(s > 0, s, 1)[:, None]
        far = np.where(w > 0, np.abs(d), 0)
        entropy = np.where(s > 0, np.log(np.where(s > 0, s, 1)) + (p * far).sum(1), 0)
        mean1, mean2 = (p * far).sum(1), (p * far * far).sum(1)
        have = (tokens >= 0) & (tokens < n)
        at = np.where(have, tokens, 0)
        own = x[np.arange(rows), at]
        logp = np.where(have, np.where(s > 0, own - lse, -np.inf), 0)
        weight = (n / 64 + 48 + 3 * mean1) * u
        size = np.where(np.isfinite(lse), np.abs(lse) + np.abs(np.log(np.where(s > 0, s, 1))), 0)
        lse_bound = weight + 3 * u * size
        logp_bound = np.where(have, weight + 3 * u * np.where(np.isfinite(own), np.abs(own - base) + size, 0), 0)
        entropy_bound = weight * (2 * mean1 + 2) + 4 * u * (mean2 + mean1 + 2 * np.abs(np.log(np.where(s > 0, s, 1))))
    return lse, logp, entropy, lse_bound, logp_bound, entropy_bound


def best(x, k):
    """Positions of the k best of each row, lower first among equals, NaN as -inf."""
    return np.argsort(-np.where(np.isnan(x), -np.inf, x), axis=1, kind="stable")[:, :k]


def close(got, want, bound):
    with np.errstate(invalid="ignore"):
        return ((got == want) | (np.abs(got - want) <= bound)).all()


def check(x, tokens, k, got):
    lse, logp, entropy, lse_bound, logp_bound, entropy_bound = oracle(x, tokens)
    g = [v.numpy() if v is not None else None for v in got]
    assert close(g[2], lse, lse_bound), "lse"
    assert close(g[0], logp, logp_bound), "log_probs"
    assert close(g[1], entropy, entropy_bound), "entropy"
    if k == 0:
        assert g[3] is None and g[4] is None
        return
    order = best(x, k)
    assert g[4].dtype == np.int32 and np.array_equal(g[4], order)
    values = np.take_along_axis(x, order, 1).astype(np.longdouble)
    with np.errstate(invalid="ignore"):
        want = np.where(np.isneginf(lse)[:, None], -np.inf, values - lse[:, None])
        bound = lse_bound[:, None] + 3 * U[x.dtype.type] * np.where(np.isfinite(want), np.abs(want) + np.abs(values), 0)
    assert close(g[3], want, bound), "top_log_probs"


def call(D, x, tokens, k):
    return D.op.token_log_probs(D.Array.from_numpy(x), D.Array.from_numpy(tokens), k)


@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_forward(gpu, D, rng, vocab, dtype):
    for rows, shift, k in ((1, 0, 5), (3, 1, 0), (9, 0, 20), (300 if vocab <= 4099 else 21, 3, 1), (70 if vocab <= 8192 else 5, 2, 64)):
        full = (rng.randn(rows, vocab + shift) * 3).astype(dtype)
        tokens = rng.randint(0, vocab, rows).astype(np.int32)
        a = D.Array.from_numpy(full)
        a = a[:, shift:] if shift else a
        k = min(k, vocab)
        check(full[:, shift:], tokens, k, D.op.token_log_probs(a, D.Array.from_numpy(tokens), k))


@pytest.mark.parametrize("vocab", [2, 40, 97, 300, 1024, 1500, 5000, 32000, 50257])
@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_masks(gpu, D, rng, vocab, dtype):
    k = min(7, vocab)
    low = np.finfo(dtype).min
    rows = 16
    x = (rng.randn(rows, vocab) * 3).astype(dtype)
    x[0] = -np.inf                                   # nothing left
    x[1] = low                                       # nothing left, by the type's lowest value
    x[2, 1:] = -np.inf                               # one left, at the front
    x[3, :-1] = -np.inf                              # one left, at the back
    x[4, rng.rand(vocab) < 0.9] = -np.inf
    x[5, rng.rand(vocab) < 0.9] = low
    x[6, :-1] = low
    x[7, vocab // 2:] = -np.inf
    x[8] = 0.0                                       # all equal
    x[9] = np.where(np.arange(vocab) % 2, 0.0, -0.0)  # equal zeros of either sign
    x[10, :] = -1e30 if dtype == np.float32 else -1e300
    x[10, vocab // 3] = 80.0
    x[11] = np.arange(vocab)[::-1]                   # sorted down and up
    x[12] = np.arange(vocab)
    x[13] = np.round(x[13])                          # many ties
    x[14, :] = np.arange(vocab) // 4                 # runs of equals, rising
    x[15, 0] = 1e30
    tokens = rng.randint(0, vocab, rows).astype(np.int32)
    for kk in sorted({0, 1, k, min(64, vocab)}):
        check(x, tokens, kk, call(D, x, tokens, kk))
    # one row at a time: the form for single tokens
    for r in range(rows):
        check(x[r:r + 1], tokens[r:r + 1], k, call(D, x[r:r + 1], tokens[r:r + 1], k))


@pytest.mark.parametrize("vocab", [97, 1500, 32000])
@pytest.mark.parametrize("rows", [1, 200])
def test_clustered_entries(gpu, D, rng, vocab, rows):
    """The best entries side by side, or all in the strides that one thread walks."""
    x = rng.randn(rows, vocab).astype(np.float32)
    for r in range(rows):
        step = [1, 4, 64, 256, 1024][r % 5]
        at = (r % 7 + np.arange(80) * step) % vocab
        x[r, at] = 50 + rng.permutation(80).astype(np.float32)
    tokens = rng.randint(0, vocab, rows).astype(np.int32)
    for k in (1, 20, 64):
        check(x, tokens, k, call(D, x, tokens, k))


@pytest.mark.parametrize("rows,vocab,stride", [(5, 4000, 256), (1, 40000, 256), (1, 1000000, 256), (600, 20000, 256), (1030, 4000, 64), (1030, 400, 64)])
@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_more_good_entries_than_are_ranked_at_once(gpu, D, rows, vocab, stride, dtype):
    """Nearly all of the best lie in the groups of few threads: `stride` groups of 16 bytes apart, in every segment."""
    rng = np.random.RandomState(vocab)
    group = np.arange(vocab) * np.dtype(dtype).itemsize // 16
    x = rng.randn(rows, vocab).astype(dtype)
    x[:, group % stride < (50 if stride == 256 else 40)] += 100
    x[:, ::7] = np.round(x[:, ::7])  # (with ties)
    tokens = rng.randint(0, vocab, rows).astype(np.int32)
    for k in (12, 20, 64):
        check(x, tokens, k, call(D, x, tokens, k))


@pytest.mark.parametrize("vocab", [5, 97, 1100, 40000])
def test_infinities_and_nan_stay_in_their_rows(gpu, D, rng, vocab):
    x = (rng.randn(8, vocab) * 3).astype(np.float32)
    x[1, 0], x[3, vocab - 1], x[5] = np.nan, np.inf, np.nan
    tokens = rng.randint(0, vocab, 8).astype(np.int32)
    k = min(9, vocab)
    got = call(D, x, tokens, k)
    bad, good = [1, 3, 5], [0, 2, 4, 6, 7]
    for v in got[:3]:
        assert np.isnan(v.numpy()[bad]).all()
    assert np.array_equal(got[4].numpy(), best(x, k))

    class Rows:
        def __init__(self, a):
            self.a = a.numpy()[good]

        def numpy(self):
            return self.a
    check(x[good], tokens[good], k, [Rows(v) for v in got])


@pytest.mark.parametrize("vocab", [1, 33, 97, 1100, 40000])
def test_rows_without_a_token(gpu, D, rng, vocab):
    x = rng.randn(6, vocab).astype(np.float32)
    tokens = np.array([0, -1, vocab - 1, vocab, 2 ** 31 - 1, -2 ** 31], np.int32)
    got = call(D, x, tokens, 1)
    check(x, tokens, 1, got)
    assert np.array_equal(got[0].numpy()[[1, 3, 4, 5]], np.zeros(4, np.float32))
    g, h = rng.randn(6).astype(np.float32), rng.randn(6).astype(np.float32)
    check_backward(D, x, tokens, g, h)
    check_backward(D, x, tokens, g, None)


def check_backward(D, x, tokens, g, h, view=None):
    u = U[x.dtype.type]
    lse, _, entropy = oracle(x, tokens)[:3]
    lse, entropy = lse.astype(x.dtype), entropy.astype(x.dtype)
    op, A = D.op, D.Array.from_numpy
    a = view if view is not None else A(x)
    got = op.token_log_probs_backward(A(g), None if h is None else A(h), a, A(tokens), A(lse), None if h is None else A(entropy)).numpy()
    x, l, e, g = (v.astype(np.longdouble) for v in (x, lse, entropy, g))
    h = np.zeros_like(g) if h is None else h.astype(np.longdouble)
    rows, n = x.shape
    empty = np.isneginf(l)
    with np.errstate(invalid="ignore", over="ignore"):
        d = x - np.where(empty, 0, l)[:, None]
        p = np.exp(d)
        far = np.where(p > 0, d, 0)
    have = (tokens >= 0) & (tokens < n) & ~empty
    g = np.where(have, g, 0)
    want = -p * (g[:, None] + h[:, None] * (far + e[:, None]))
    want[np.arange(rows)[have], tokens[have]] += g[have]
    parts = np.abs(g)[:, None] + np.abs(h)[:, None] * (np.abs(far) + np.abs(e)[:, None])
    bound = p * parts * (4 * np.abs(far) + 12) * u
    bound[np.arange(rows)[have], tokens[have]] += 2 * u * np.abs(g[have])
    assert got.shape == want.shape and (np.abs(got - want) <= bound + np.finfo(got.dtype).tiny * (1 + parts)).all()
    return got


@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_backward(gpu, D, rng, vocab, dtype):
    for rows, shift in ((1, 0), (3, 1), (300 if vocab <= 4099 else 9, 0), (50 if vocab <= 8192 else 5, 3)):
        full = (rng.randn(rows, vocab + shift) * 3).astype(dtype)
        tokens = rng.randint(0, vocab, rows).astype(np.int32)
        g, h = rng.randn(rows).astype(dtype), rng.randn(rows).astype(dtype)
        a = D.Array.from_numpy(full)
        check_backward(D, full[:, shift:], tokens, g, h, a[:, shift:] if shift else a)
        check_backward(D, full[:, shift:], tokens, g, None, a[:, shift:] if shift else a)


@pytest.mark.parametrize("vocab", [2, 97, 1500, 32000])
def test_backward_of_masked_rows(gpu, D, rng, vocab):
    x = (rng.randn(8, vocab) * 3).astype(np.float32)
    x[0] = -np.inf
    x[1] = np.finfo(np.float32).min
    x[2, 1:] = -np.inf
    x[3, rng.rand(vocab) < 0.9] = -np.inf
    x[4, :-1] = np.finfo(np.float32).min
    x[5, 0] = 1e30
    tokens = rng.randint(0, vocab, 8).astype(np.int32)
    g, h = rng.randn(8).astype(np.float32), rng.randn(8).astype(np.float32)
    got = check_backward(D, x, tokens, g, h)
    assert not got[0].any()


@pytest.mark.parametrize("vocab", [40, 1500, 9000])
def test_large_gradients_of_masked_rows(gpu, D, rng, vocab):
    """A masked entry's gradient is 0 whatever comes from above (but for the given token's own part, which does not ask for its probability)."""
    x = rng.randn(5, vocab).astype(np.float32)
    x[:4, rng.rand(vocab) < 0.5] = -np.inf
    x[2] = -np.inf
    x[3, 1:] = np.finfo(np.float32).min
    x[:2, 0] = x[4, 0] = 1.0
    g, h = np.array([1e30, -1e30, 1e30, 1e20, 0], np.float32), np.array([1e30, 1e32, -1e30, 1e30, 1e30], np.float32)
    got = check_backward(D, x, np.zeros(5, np.int32), g, h)
    assert (got[:, 1:][np.isneginf(x[:, 1:])] == 0).all()


@pytest.mark.parametrize("vocab", [2, 97, 1500, 9000])
def test_gradient_against_differences(gpu, D, rng, vocab):
    rows, step = 3, 1e-5
    x = rng.randn(rows, vocab) * 2
    tokens = rng.randint(0, vocab, rows).astype(np.int32)
    g, h = rng.randn(rows), rng.randn(rows)
    A = D.Array.from_numpy

    def loss(x):
        r = call(D, x, tokens, 0)
        return float((r[0].numpy() * g + r[1].numpy() * h).sum())

    _, entropy, lse, _, _ = call(D, x, tokens, 0)
    grad = D.op.token_log_probs_backward(A(g), A(h), A(x), A(tokens), lse, entropy).numpy()
    along = rng.randn(rows, vocab)
    slope = (loss(x + step * along) - loss(x - step * along)) / (2 * step)
    # third derivatives are of the size of the logits' own spread cubed, and the loss is rounded at 1e-16 of some tens
    assert abs(slope - (grad * along).sum()) <= 1e3 * step ** 2 * (np.abs(g) + np.abs(h)).sum() * 10 + 1e-14 * 100 / step


def test_shapes_and_views(gpu, D, rng):
    x = (rng.randn(3, 4, 50, 97) * 3).astype(np.float32)
    a = D.Array.from_numpy(x)
    for view, ref in ((a, x), (a[:, 1], x[:, 1]), (a[::2, :, ::-1], x[::2, :, ::-1]), (a.transpose(1, 0, 2, 3), x.transpose(1, 0, 2, 3)),
                      (a.transpose(0, 1, 3, 2), x.transpose(0, 1, 3, 2)), (a[:, :, :, 5:], x[..., 5:]), (a[0, 0, 0], x[0, 0, 0])):
        lead, n = ref.shape[:-1], ref.shape[-1]
        tokens = np.asarray(rng.randint(0, n, lead)).astype(np.int32)
        # (numpy's contiguous form of a single number has one axis)
        got = D.op.token_log_probs(view, D.Array.from_numpy(tokens).reshape(lead), 3)
        assert [v.shape for v in got] == [lead, lead, lead, lead + (3,), lead + (3,)]

        class Flat:
            def __init__(self, v, k):
                self.a = v.numpy().reshape((-1, 3) if k else (-1,))

            def numpy(self):
                return self.a
        flat = np.ascontiguousarray(ref).reshape(-1, n)
        check(flat, tokens.reshape(-1), 3, [Flat(v, i > 2) for i, v in enumerate(got)])


@pytest.mark.parametrize("rows,vocab", [(0, 7), (1, 50257), (64, 97), (30, 5000)])
def test_destinations(gpu, D, rng, rows, vocab):
    op, A = D.op, D.Array.from_numpy
    x, tokens = rng.randn(rows, vocab).astype(np.float32), rng.randint(0, vocab, rows).astype(np.int32)
    want = call(D, x, tokens, 4)
    out = [D.Array.empty((rows,)) for _ in range(3)] + [D.Array.empty((rows, 4)), D.Array.empty((rows, 4), D.DTYPE_INT32)]
    got = op.token_log_probs(A(x), A(tokens), 4, out=out)
    assert all(p is q for p, q in zip(got, out)) and all(np.array_equal(p.numpy(), q.numpy()) for p, q in zip(got, want))
    g = A(rng.randn(rows).astype(np.float32))
    a = A(x)
    d = op.token_log_probs_backward(g, g, a, A(tokens), want[2], want[1])
    assert np.array_equal(a.numpy(), x)
    assert op.token_log_probs_backward(g, g, a, A(tokens), want[2], want[1], out=a) is a
    assert np.array_equal(a.numpy(), d.numpy())


def test_results_that_repeat(gpu, D, rng):
    for rows, vocab in ((1, 50257), (5, 32000), (900, 32000), (4000, 97)):
        x, tokens = np.round(rng.randn(rows, vocab) * 3, 2).astype(np.float32), rng.randint(0, vocab, rows).astype(np.int32)
        a, t = D.Array.from_numpy(x), D.Array.from_numpy(tokens)
        first = [v.numpy() for v in D.op.token_log_probs(a, t, 20)]
        for _ in range(5):
            assert all(np.array_equal(p, q.numpy()) for p, q in zip(first, D.op.token_log_probs(a, t, 20)))


def test_recorded(gpu, D, rng):
    op = D.op
    for rows, vocab in ((1, 50257), (40, 3000), (70, 97)):
        x, tokens = D.Array.from_numpy(rng.randn(rows, vocab).astype(np.float32)), D.Array.from_numpy(rng.randint(0, vocab, rows).astype(np.int32))
        g = D.Array.from_numpy(rng.randn(rows).astype(np.float32))
        fill = D.Array.empty((rows, vocab))
        fill.assign(x)
        with D.Recording() as rec:
            got = op.token_log_probs(fill, tokens, 5)
            got += (op.token_log_probs_backward(g, g, fill, tokens, got[2], got[1]),)
        for graph in (False, True):
            if graph:
                rec.make_graph()
            for step in range(3):
                fill.assign(x * float(step + 2))
                rec.replay()
                want = op.token_log_probs(fill, tokens, 5)
                want += (op.token_log_probs_backward(g, g, fill, tokens, want[2], want[1]),)
                assert all(np.array_equal(p.numpy(), q.numpy()) for p, q in zip(got, want)), (graph, step)


def test_device_refusals(gpu, D, rng):
    op, A = D.op, D.Array.from_numpy
    buf = A(rng.randn(16, 32).astype(np.float32))
    before, tokens = buf.numpy(), A(np.zeros(8, np.int32))
    with pytest.raises(D.DaliError, match="entropy overlaps logits"):
        op.token_log_probs(buf[:8], tokens, out=(None, buf[3, :8], None, None, None))
    with pytest.raises(D.DaliError, match="log_probs and lse overlap"):
        op.token_log_probs(A(before[:8]), tokens, out=(buf[0, :8], None, buf[0, 4:12], None, None))
    one = A(np.ones(8, np.float32))
    with pytest.raises(D.DaliError, match="d_logits overlaps logits"):
        op.token_log_probs_backward(one, None, buf[:8], tokens, one, None, out=buf[1:9])
    assert np.array_equal(buf.numpy(), before)


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("rows,vocab", [(7, 5), (9, 97), (5, 300), (1030, 1300), (300, 3001), (2, 50257), (140, 12345)])
def test_an_alternative_has_the_given_tokens_log_probability(gpu, D, rng, rows, vocab, dtype):
    # rows far from 0, where a difference to lse would lose digits that the difference to the maximum keeps
    x = (rng.randint(-64, 64, (rows, vocab)) / 16.0 + 30000.0).astype(dtype)
    k = 5
    order = best(x, k)
    X = D.Array.from_numpy(x)
    for place in range(k):
        tokens = np.ascontiguousarray(order[:, place]).astype(np.int32)
        log_probs, _, _, top, top_tokens = D.op.token_log_probs(X, D.Array.from_numpy(tokens), k)
        assert np.array_equal(top_tokens.numpy()[:, place], tokens)
        assert np.array_equal(top.numpy()[:, place], log_probs.numpy())

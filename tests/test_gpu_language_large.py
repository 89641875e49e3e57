"""Operators of language models on arrays whose bytes pass 2^32: the last rows of a large array against the same rows among few, bit for bit."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def with_last_rows(D, rows, last):
    """zeros [rows, width], the last of them given"""
    big = D.Array.zeros((rows, last.shape[1]))
    big[rows - last.shape[0]:].assign(D.Array.from_numpy(last))
    return big


@pytest.mark.parametrize("width", [97, 4096, 20000])
def test_layer_norm(gpu, D, rng, width):
    rows, n = 1100000000 // width, 5
    assert rows * width * 4 > 2 ** 32
    last, dlast = (rng.randn(n, width) * 2 + 0.5).astype(np.float32), rng.randn(n, width).astype(np.float32)
    x, dy = with_last_rows(D, rows, last), with_last_rows(D, rows, dlast)
    gamma, beta = D.Array.from_numpy((1 + 0.1 * rng.randn(width)).astype(np.float32)), D.Array.from_numpy(rng.randn(width).astype(np.float32))
    want = D.op.layer_norm(D.Array.from_numpy(last), gamma, beta)
    y, mean, rstd = D.op.layer_norm(x, gamma, beta)
    assert np.array_equal(y[rows - n:].ascontiguousarray().numpy(), want[0].numpy())
    assert np.array_equal(y[rows - n - 1].ascontiguousarray().numpy(), beta.numpy())  # (a row of zeros)
    assert np.array_equal(mean.numpy()[-n:], want[1].numpy()) and np.array_equal(rstd.numpy()[-n:], want[2].numpy())
    want = D.op.layer_norm_backward(D.Array.from_numpy(dlast), D.Array.from_numpy(last), want[1], want[2], gamma)
    dx, dgamma, dbeta = D.op.layer_norm_backward(dy, x, mean, rstd, gamma, out=(y, None, None))
    assert np.array_equal(dx[rows - n:].ascontiguousarray().numpy(), want[0].numpy())
    # (sums of five rows among zeros, in another order; a normalised value is below 8)
    for got, ref, size in ((dgamma, want[1], np.abs(dlast) * 8), (dbeta, want[2], np.abs(dlast))):
        assert (np.abs(got.numpy() - ref.numpy()) <= 10 * 2.0 ** -24 * size.sum(0)).all()


@pytest.mark.parametrize("vocab", [97, 5000, 50257])
def test_token_log_probs(gpu, D, rng, vocab):
    rows, n, k = 1100000000 // vocab, 5, 6
    last = (rng.randn(n, vocab) * 3).astype(np.float32)
    x = with_last_rows(D, rows, last)
    tokens = np.zeros(rows, np.int32)
    tokens[-n:] = rng.randint(0, vocab, n)
    small, t = D.Array.from_numpy(last), D.Array.from_numpy(tokens)
    # (few rows may be summed in another order: the same rows among 1100, which take the form for many)
    some = np.zeros((1100, vocab), np.float32)
    some[-n:] = last
    some_tokens = np.zeros(1100, np.int32)
    some_tokens[-n:] = tokens[-n:]
    want = D.op.token_log_probs(D.Array.from_numpy(some), D.Array.from_numpy(some_tokens), k)
    got = D.op.token_log_probs(x, t, k)
    for g, w in zip(got, want):
        assert np.array_equal(g.numpy()[-n - 1:], w.numpy()[-n - 1:])
    g = np.zeros(rows, np.float32)
    g[-n:] = rng.randn(n)
    entropy, lse = got[1], got[2]
    dg, dg_small = D.Array.from_numpy(g), D.Array.from_numpy(g[-n:])
    want = D.op.token_log_probs_backward(dg_small, dg_small, small, D.Array.from_numpy(tokens[-n:]), D.Array.from_numpy(lse.numpy()[-n:]), D.Array.from_numpy(entropy.numpy()[-n:]))
    d = D.op.token_log_probs_backward(dg, dg, x, t, lse, entropy, out=x)
    assert np.array_equal(d[rows - n:].ascontiguousarray().numpy(), want.numpy())
    assert not d[rows - n - 1].ascontiguousarray().numpy().any()


def test_clip_by_global_norm(gpu, D, rng):
    rows, width = 270000, 4097
    last, other = rng.randn(3, width).astype(np.float32), rng.randn(1000).astype(np.float32)
    a, b = with_last_rows(D, rows, last), D.Array.from_numpy(other)
    norm = np.sqrt((last.astype(np.float64) ** 2).sum() + (other.astype(np.float64) ** 2).sum())
    got, n = D.op.clip_by_global_norm([a, b], 1.0, out=([a, b], None))
    assert abs(float(n.numpy()) - norm) <= norm * 2.0 ** -23
    for g, w in ((got[0][rows - 3:].ascontiguousarray().numpy(), last / norm), (got[1].numpy(), other / norm)):
        assert (np.abs(g - w) <= 3 * 2.0 ** -24 * np.abs(w)).all()
    assert not got[0][rows - 4].ascontiguousarray().numpy().any()

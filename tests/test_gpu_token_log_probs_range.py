"""Log probabilities of tokens and their gradient near the ends of their types' range, and of rows far from 0. u is half a unit in the last place of 1."""
import numpy as np
import pytest

from test_gpu_token_log_probs import U, best, check_backward

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [40, 97, 1500, 9000])
@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_gradients_at_the_end_of_the_range(gpu, D, rng, vocab, dtype):
    """A masked entry's gradient is 0, and that of an improbable one a finite number, up to the largest gradient from above."""
    big = np.finfo(dtype).max
    x = (rng.randn(6, vocab) * 3).astype(dtype)
    x[:, rng.rand(vocab) < 0.5] = -np.inf
    x[2, 1:] = np.finfo(dtype).min
    x[3] = -np.inf
    x[:3, 0] = x[4:, 0] = 1.0
    x[4, 1:9] = -np.arange(8) * 12  # (improbable, not masked)
    h = (big * np.array([0.9, -0.5, 0.2, 0.9, 0.01, 0])).astype(dtype)
    g = (big * np.array([0.1, 0.1, -0.3, 0.5, -0.01, 0.9])).astype(dtype)
    lowest = np.isneginf(x) | (x == np.finfo(dtype).min)
    for up in (h / dtype(64), h):
        got = check_backward(D, x, np.zeros(6, np.int32), g if up is not h else g * 0, up)
        assert not got[lowest & (np.arange(vocab) > 0)].any() and np.isfinite(got[:, 0]).all()


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("rows,vocab", [(7, 5), (9, 97), (5, 300), (1030, 1300), (300, 3001), (2, 50257), (140, 12345)])
def test_log_probabilities_of_rows_far_from_0(gpu, D, rng, rows, vocab, dtype):
    """They are differences to the row's maximum: the size of the logits costs them nothing."""
    u, k = U[dtype], 5
    x = (rng.randint(-64, 64, (rows, vocab)) / 16.0 + 30000.0).astype(dtype)  # (exact in both types)
    tokens = rng.randint(0, vocab, rows).astype(np.int32)
    log_probs, entropy, _, top, top_tokens = (v.numpy() for v in D.op.token_log_probs(D.Array.from_numpy(x), D.Array.from_numpy(tokens), k))
    d = x.astype(np.longdouble) - x.max(1, keepdims=True)
    w = np.exp(d)
    ln = np.log(w.sum(1))
    far = (w * -d).sum(1) / w.sum(1)
    # the sum's error as in test_gpu_token_log_probs.py, then the logarithm and two differences
    bound = (vocab / 64 + 48 + 3 * far) * u + 3 * u * ln
    own = d[np.arange(rows), tokens]
    assert (np.abs(log_probs - (own - ln)) <= bound + 3 * u * np.abs(own)).all()
    order = best(x, k)
    values = np.take_along_axis(d, order, 1)
    assert np.array_equal(top_tokens, order)
    assert (np.abs(top - (values - ln[:, None])) <= bound[:, None] + 3 * u * np.abs(values)).all()

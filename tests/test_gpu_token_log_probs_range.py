"""Log probabilities of tokens and their gradient near the ends of their types' range. u is half a unit in the last place of 1."""
import numpy as np
import pytest

from test_gpu_token_log_probs import check_backward

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

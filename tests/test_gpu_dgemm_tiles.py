"""fp64 products with large and small tiles (128 x 128 where they come in nearly whole rounds of two to a compute unit, 256 of them), on whole numbers, whose sums are exact."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


# 512 large tiles, 480 (the fewest of a round), 475, 1005 of two rounds with ragged ends; small ones; a row and a column
@pytest.mark.parametrize("M,N,K", [(4096, 2048, 37), (4096, 1920, 16), (2432, 3200, 20), (8572, 1910, 33), (2049, 2050, 35), (130, 70, 300), (1, 4000, 50), (4000, 1, 50)])
@pytest.mark.parametrize("ta,tb", [(0, 0), (1, 0), (0, 1), (1, 1)])
def test_tiles(gpu, D, rng, M, N, K, ta, tb):
    a, b = (rng.randint(-9, 10, s).astype(np.float64) for s in ((M, K), (K, N)))
    A = lambda x, t: D.Array.from_numpy(np.ascontiguousarray(x.T)).T if t else D.Array.from_numpy(x)  # noqa: E731
    assert np.array_equal(D.op.dot(A(a, ta), A(b, tb)).numpy(), a @ b)

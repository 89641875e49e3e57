"""The global norm of doubles whose squares are no doubles, and clipping by it."""
import numpy as np
import pytest

from test_gpu_global_norm import reference

pytestmark = pytest.mark.gpu


def check_clipped(D, arrays, max_norm):
    """The bounds of test_gpu_global_norm.py; a result below the smallest normal number is rounded to a multiple of the smallest one of all, the norm too."""
    u, tiny = 2.0 ** -53, np.finfo(np.float64).smallest_subnormal
    held = [D.Array.from_numpy(a) for a in arrays]
    got, norm = D.op.clip_by_global_norm(held, max_norm)
    want, wnorm = reference(arrays, max_norm)
    loss = sum(a.size for a in arrays) * u + 4 * u
    for n in (norm, D.op.global_norm(held)):
        assert abs(n.numpy() - wnorm) <= wnorm * (loss + u) + tiny
    for a, g, w in zip(arrays, got, want):
        if wnorm <= max_norm * (1 - 1e-6):
            assert np.array_equal(g.numpy(), a)
        else:
            assert (np.abs(g.numpy() - w) <= np.abs(w) * (2.5 * u + loss) + tiny).all()


@pytest.mark.parametrize("sizes", [[1], [7], [100, 33], [5000], [9000, 17], [300000, 5], [1 << 20, 3, 70001], [11] * 40, [4001] * 100])
def test_norms_of_doubles_whose_squares_pass_the_range(gpu, D, rng, sizes):
    """Squares of values above 1.3e154 are no doubles, those of values below 1.5e-162 are 0; the norm and the clipped arrays are ordinary numbers."""
    for size in (1e200, 1e-200, 1e300, 1e-300, 1e153, 1e-161, 1e-310):
        arrays = [rng.randn(n) * size for n in sizes]
        length = np.sqrt(sum(sizes))
        for max_norm in (size * length / 7, size * length * 7):
            check_clipped(D, arrays, max_norm)
    for size in (1e200, 1e300):
        check_clipped(D, [rng.randn(n) * size for n in sizes], 1.0)
        check_clipped(D, [rng.randn(n) * size for n in sizes], 1e-20)
    # side by side: large, ordinary and small ones, and numbers near where one kind ends and the next begins
    mixed = [rng.randn(n) * 10.0 ** rng.choice([-310, -250, -200, -150, -140, 0, 100, 140, 150, 155, 200], n) for n in sizes]
    check_clipped(D, mixed, 1.0)
    for top in (-150, -140, 0, 140, 150):
        check_clipped(D, [rng.randn(n) * 10.0 ** rng.uniform(top - 20, top, n) for n in sizes], 10.0 ** (top - 5))


@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("n", [5, 3000, 300000])
def test_a_norm_of_doubles_that_is_not_finite(gpu, D, rng, value, n):
    for size in (1.0, 1e200, 1e-200):
        arrays = [rng.randn(n) * size, rng.randn(17)]
        arrays[0][n // 2] = value
        got, got_norm = D.op.clip_by_global_norm([D.Array.from_numpy(a) for a in arrays], 0.1)
        assert np.isnan(got_norm.numpy()) if np.isnan(value) else np.isinf(got_norm.numpy())
        assert all(np.array_equal(g.numpy(), a, equal_nan=True) for g, a in zip(got, arrays))
    # (finite values whose norm passes the type's range)
    arrays = [np.full(n, 1.7e308), np.full(17, 1.0)]
    got, got_norm = D.op.clip_by_global_norm([D.Array.from_numpy(a) for a in arrays], 0.1)
    assert np.isinf(got_norm.numpy()) and all(np.array_equal(g.numpy(), a) for g, a in zip(got, arrays))


@pytest.mark.parametrize("n", [1, 7, 3000, 300000])
@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_a_largest_norm_of_0(gpu, D, rng, n, dtype):
    """Everything is scaled to 0, however small it is."""
    for size in {np.float32: [1.0, 1e-44, 1e38], np.float64: [1.0, 1e-150, 1e-200, 1e-320, 1e300]}[dtype]:
        a = np.abs(rng.randn(n)) + 1
        got, norm = D.op.clip_by_global_norm([D.Array.from_numpy((a / a.max() * size).astype(dtype))], 0.0)
        assert norm.numpy() > 0 and not got[0].numpy().any()

"""Layer normalisation over the whole range of its types: rows whose squares or sums pass it, rows without spread at any size. u is half a unit in the last place of 1;
`depth` of test_gpu_layer_norm.py bounds the roundings of a sum."""
import numpy as np
import pytest

from test_gpu_layer_norm import U, backward_bounds, depth, oracle

pytestmark = pytest.mark.gpu

WIDTHS = [1, 3, 8, 31, 64, 97, 128, 250, 256, 512, 1000, 1024, 2047, 4096, 5000, 8192, 16384, 20000, 31000, 32768, 50001]
CONSTANTS = {np.float32: [0.1, -3.3, 1e10, 1.7e19, -1e24, 1e27, -1e30, 3e38, np.finfo(np.float32).max, -np.finfo(np.float32).max, 1e-30, 1e-44],
             np.float64: [0.1, -3.3, 1e10, 1e100, -1e154, 1e170, -1e200, 1.7e308, np.finfo(np.float64).max, -np.finfo(np.float64).max, 1e-200, 5e-324]}


def norm(D, x, gamma=None, beta=None, epsilon=1e-5):
    a = D.Array.from_numpy
    return [v.numpy() for v in D.op.layer_norm(a(x), None if gamma is None else a(gamma), None if beta is None else a(beta), epsilon)]


def check(x, gamma, beta, epsilon, got):
    """The bounds of test_gpu_layer_norm.py, with the values' sizes summed where they do not pass the range"""
    u = U[x.dtype.type]
    y, mean, rstd = got
    want, wmean, wrstd = oracle(x, gamma, beta, epsilon)
    tol = (depth(x.shape[-1]) + 16) * u
    spread, size = np.abs(x - wmean[..., None]).mean(-1), np.abs(x.astype(np.longdouble)).mean(-1)
    assert (np.abs(mean - wmean) <= u * np.abs(wmean) + tol * spread + tol * u * size).all()
    lost = (tol * tol * size + tol * spread) * wrstd
    assert (np.abs(rstd - wrstd) <= wrstd * (tol + lost * lost)).all()
    unit = np.abs((want - beta) / np.where(gamma == 0, 1, gamma))
    bound = np.abs(gamma) * (lost[..., None] + (tol + (lost * lost)[..., None]) * unit) + 2 * u * (np.abs(beta) + np.abs(want))
    assert np.isfinite(bound).all() and (np.abs(y - want) <= bound).all()


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_rows_of_one_value(gpu, D, rng, width, dtype):
    """The mean is the value, the distances from it are 0: y is beta, bit for bit, and rstd that of epsilon."""
    values = np.array(CONSTANTS[dtype], dtype)
    x = np.repeat(values[:, None], width, 1)
    gamma, beta = (1 + rng.randn(width)).astype(dtype), rng.randn(width).astype(dtype)
    y, mean, rstd = norm(D, x, gamma, beta)
    assert np.array_equal(y, np.repeat(beta[None], len(values), 0))
    assert np.array_equal(mean, values)
    # (one rounding each of epsilon, the root and the quotient)
    np.testing.assert_allclose(rstd, 1 / np.sqrt(np.longdouble(1e-5)), rtol=4 * U[dtype])


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_large_values(gpu, D, rng, width, dtype):
    """The normalised row does not depend on the size of its values, whether their squares and sums fit the type or not."""
    gamma, beta = (1 + 0.2 * rng.randn(width)).astype(dtype), (0.2 * rng.randn(width)).astype(dtype)
    for size in {np.float32: [1e15, 1e18, 1e21, 1e30, 1e37], np.float64: [1e140, 1e152, 1e160, 1e250, 1e307]}[dtype]:
        for offset in (0.3, 5.0):
            x = ((np.clip(rng.randn(7, width), -5, 5) / 2 + offset) * size).astype(dtype)
            check(x, gamma, beta, 1e-5, norm(D, x, gamma, beta))


@pytest.mark.parametrize("width", [2, 3, 64, 250, 1024, 5000, 20000, 50001])
@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_rows_at_the_ends_of_the_range(gpu, D, rng, width, dtype):
    """Largest and lowest values in one row: their distance passes the type's range."""
    big, u = np.finfo(dtype).max, U[dtype]
    x = np.where(rng.rand(5, width) < 0.5, big, -big).astype(dtype)
    x[:, 0], x[:, 1] = big, -big
    y, mean, rstd = norm(D, x)
    want, wmean, wrstd = oracle(x, np.ones(width, dtype), np.zeros(width, dtype), 1e-5)
    tol = (depth(width) + 16) * u
    assert (np.abs(mean - wmean) <= tol * big).all()
    # (rstd is below the smallest normal number)
    assert (np.abs(rstd - wrstd) <= tol * wrstd + np.finfo(dtype).smallest_subnormal).all()
    assert (np.abs(y - want) <= 4 * tol * (1 + np.abs(want)) * (1 + np.abs(wmean) * wrstd)[:, None]).all()


@pytest.mark.parametrize("width", [3, 31, 64, 250, 1000, 4096, 5000, 20000, 50001])
@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_rows_that_differ_in_their_last_places(gpu, D, rng, width, dtype):
    """Far from 0, a few units in the last place apart: the distances are exact once the mean is, whatever it was rounded to at first."""
    u = U[dtype]
    for size in {np.float32: [1.0, 1e6, 1e24, 1e30], np.float64: [1.0, 1e6, 1e160, 1e200]}[dtype]:
        steps = rng.randint(-3, 4, (6, width))
        steps[:, 0], steps[:, 1] = -3, 3
        base = dtype(2.0) ** np.floor(np.log2(dtype(size))) * dtype(1.5)
        x = (base + steps * (np.spacing(base))).astype(dtype)
        y, mean, rstd = norm(D, x, epsilon=0.0)
        # (from the steps: a mean of the values themselves, in whatever precision, loses what they differ in)
        middle, apart = steps.astype(np.longdouble).mean(1), np.longdouble(np.spacing(base))
        away = steps - middle[:, None]
        wmean, wrstd = base + middle * apart, 1 / (np.sqrt((away * away).mean(1)) * apart)
        want = away * apart * wrstd[:, None]
        assert (np.abs(mean - wmean) <= 2 * u * np.abs(wmean)).all()
        # sums of distances (as many units as the first mean is off) and of their squares are off by depth * u of their terms
        tol = (depth(width) + 16) * u
        assert (np.abs(rstd - wrstd) <= 4 * tol * wrstd).all()
        assert (np.abs(y - want) <= 4 * tol * (np.abs(want) + depth(width))).all()


@pytest.mark.parametrize("width", [5, 31, 64, 97, 128, 250, 1024, 5000])
def test_a_row_does_not_depend_on_the_others(gpu, D, rng, width):
    """Rows that share a wave or a workgroup, some with values that their neighbours do not have."""
    x = rng.randn(70, width).astype(np.float32)
    alone = [np.concatenate(v) for v in zip(*[norm(D, x[r:r + 1]) for r in range(70)])]
    odd = x.copy()
    odd[1::5], odd[2::5, 0], odd[3::5, -1], odd[14::20] = -1e30, np.inf, np.nan, 3e37 * x[14::20]
    same = np.isin(np.arange(70) % 5, [0, 4]) & (np.arange(70) % 20 != 14)
    for p, q, r in zip(norm(D, x), norm(D, odd), alone):
        assert np.array_equal(p, r) and np.array_equal(q[same], r[same])
    assert not norm(D, odd)[0][1::5].any()
    place = D.Array.from_numpy(odd)
    D.op.layer_norm(place, out=(place, None, None))
    assert np.array_equal(place.numpy(), norm(D, odd)[0], equal_nan=True)


@pytest.mark.parametrize("width", [2, 3, 64, 97, 250, 1024, 5000, 20000, 50001])
@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_gradient_at_the_ends_of_the_range(gpu, D, rng, width, dtype):
    """x - mean passes the type's range where x does not; u = (x - mean) rstd is an ordinary number."""
    big, u, rows = np.finfo(dtype).max, U[dtype], 40
    x = np.where(rng.rand(rows, width) < 0.2, big, -big).astype(dtype)
    x[:, 0], x[:, 1] = big, -big
    x[1::2] *= dtype(0.2)
    dy, gamma = rng.randn(rows, width).astype(dtype), (1 + 0.2 * rng.randn(width)).astype(dtype)
    _, mean, rstd = (v.astype(dtype) for v in oracle(x, gamma, 0 * gamma, 1e-5))
    got = [v.numpy() for v in D.op.layer_norm_backward(*[D.Array.from_numpy(v) for v in (dy, x, mean, rstd, gamma)])]
    # (the statistics are operands: what they were rounded to is not the kernel's error)
    for g, (want, bound) in zip(got, backward_bounds(dy, x, mean, rstd, gamma)):
        assert np.isfinite(bound.astype(dtype)).all()
        assert (np.abs(g - want) <= bound + 4 * np.finfo(dtype).smallest_subnormal).all()

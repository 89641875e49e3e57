"""The norm over many arrays and clipping by it, against sums in higher precision: sizes, counts, values at the ends of the range, destinations."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = {np.float32: 2.0 ** -24, np.float64: 2.0 ** -53}


def reference(arrays, max_norm):
    norm = np.sqrt(sum((a.astype(np.longdouble) ** 2).sum() for a in arrays))
    return [a.astype(np.longdouble) * (max_norm / norm if norm > max_norm else 1) for a in arrays], norm


def check(D, arrays, max_norm, out=None):
    u = U[arrays[0].dtype.type]
    held = [D.Array.from_numpy(a) for a in arrays]
    got, norm = D.op.clip_by_global_norm(held, max_norm, out=out)
    want, wnorm = reference(arrays, max_norm)
    count = sum(a.size for a in arrays)
    # summed in double: at most `count` roundings of 2^-53, halved by the square root, then one to the type
    loss = count * 2.0 ** -53 + 4 * 2.0 ** -53
    for n in (norm, D.op.global_norm(held)):
        assert n.shape == ()
        # (a norm that passes the type's range is reported as inf)
        assert abs(n.numpy() - wnorm) <= wnorm * (loss + u) if wnorm <= np.finfo(arrays[0].dtype).max else np.isinf(n.numpy())
    tiny = np.finfo(arrays[0].dtype).smallest_subnormal
    for a, g, w in zip(arrays, got, want):
        assert g.shape == a.shape and g.dtype == D.array._FROM_NP[a.dtype]
        if wnorm <= max_norm * (1 - 1e-6):
            assert np.array_equal(g.numpy(), a)
        else:
            assert (np.abs(g.numpy() - w) <= np.abs(w) * (2.5 * u + loss) + tiny).all()
    for h, a in zip(held, arrays):
        assert np.array_equal(h.numpy(), a)


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("sizes", [[1], [2], [3], [4, 5], [255], [256, 257], [1023, 1, 1025], [4096], [4097, 3], [65535], [100003, 17, 64], [1 << 20, 5, (1 << 20) + 3], [3000001], [9000001, 77]])
def test_sizes(gpu, D, rng, sizes, dtype):
    arrays = [rng.randn(n).astype(dtype) for n in sizes]
    norm = math.sqrt(sum(sizes))
    for max_norm in (norm / 7, norm * 7, float("inf")):
        check(D, arrays, max_norm)


@pytest.mark.parametrize("count", [1, 2, 30, 95, 96, 97, 192, 193, 500])
def test_many_arrays(gpu, D, rng, count):
    arrays = [rng.randn(*s).astype(np.float32) for s in [(rng.randint(1, 40), rng.randint(1, 300)) if i % 3 else (rng.randint(1, 50),) for i in range(count)]]
    check(D, arrays, 1.5)
    check(D, arrays, 1e9)


def test_empty_arrays_and_zeros(gpu, D):
    empty, zero, one = np.zeros((0, 5), np.float32), np.zeros(700, np.float32), np.full(3, 2, np.float32)
    for arrays in ([empty], [empty, empty], [zero], [empty, one, empty], [one, empty, zero], [empty] * 200 + [one]):
        for max_norm in (0.5, 100.0):
            check(D, arrays, max_norm)
    got, norm = D.op.clip_by_global_norm([D.Array.from_numpy(one)], 0.0)
    assert np.array_equal(got[0].numpy(), np.zeros(3)) and abs(norm.numpy() - math.sqrt(12)) < 1e-6
    got, norm = D.op.clip_by_global_norm([D.Array.from_numpy(zero)], 0.0)
    assert np.array_equal(got[0].numpy(), zero) and norm.numpy() == 0


def test_values_at_the_ends_of_the_range(gpu, D, rng):
    large = (rng.rand(5000) * 1e37 + 1e37).astype(np.float32)
    check(D, [large, large[:7]], 1.0)  # (neither their squares nor their norm fit a float)
    check(D, [large[:100], large[:7]], 1.0)  # (their norm does)
    small = (rng.rand(5000) * 1e-30).astype(np.float32)
    check(D, [small], 1e-32)
    # the norm itself passes the type's range: reported as inf, scaled by what it is
    huge = np.full(100, 3e38, np.float32)
    got, norm = D.op.clip_by_global_norm([D.Array.from_numpy(huge)], 1.0)
    assert np.isinf(norm.numpy())
    np.testing.assert_allclose(got[0].numpy(), np.full(100, 0.1, np.float32), rtol=1e-6)


@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("n", [5, 3000, 300000])
def test_a_norm_that_is_not_finite_scales_nothing(gpu, D, rng, value, n):
    arrays = [rng.randn(n).astype(np.float32), rng.randn(17).astype(np.float32)]
    arrays[0][n // 2] = value
    got, norm = D.op.clip_by_global_norm([D.Array.from_numpy(a) for a in arrays], 0.1)
    assert np.isnan(norm.numpy()) if np.isnan(value) else np.isinf(norm.numpy())
    assert all(np.array_equal(g.numpy(), a, equal_nan=True) for g, a in zip(got, arrays))


@pytest.mark.parametrize("n", [7, 5000, 2000003])
def test_destinations(gpu, D, rng, n):
    arrays = [rng.randn(n).astype(np.float32), rng.randn(33, 3).astype(np.float32)]
    held = [D.Array.from_numpy(a) for a in arrays]
    want, norm = D.op.clip_by_global_norm(held, 0.25)
    kept = D.Array.empty(())
    got, into = D.op.clip_by_global_norm(held, 0.25, out=(held, kept))
    assert into is kept and all(p is q for p, q in zip(got, held))
    assert np.array_equal(kept.numpy(), norm.numpy()) and all(np.array_equal(p.numpy(), q.numpy()) for p, q in zip(held, want))
    held = [D.Array.from_numpy(a) for a in arrays]
    beside = D.Array.empty((33, 3))
    got, _ = D.op.clip_by_global_norm(held, 0.25, out=([None, beside], None))
    assert got[1] is beside and all(np.array_equal(p.numpy(), q.numpy()) for p, q in zip(got, want))
    assert all(np.array_equal(h.numpy(), a) for h, a in zip(held, arrays))


def test_views_and_neighbours(gpu, D, rng):
    """Arrays that lie side by side in one buffer, at odd offsets, clipped in place; a strided one is laid out first."""
    buf = rng.randn(1001).astype(np.float32)
    a = D.Array.from_numpy(buf)
    parts = [a[1:8], a[8:500], a[500:501], a[503:1001]]
    want, _ = reference([buf[1:8], buf[8:500], buf[500:501], buf[503:1001]], 2.0)
    D.op.clip_by_global_norm(parts, 2.0, out=(parts, None))
    got = a.numpy()
    assert np.array_equal(got[[0, 501, 502]], buf[[0, 501, 502]])
    for (lo, hi), w in zip(((1, 8), (8, 500), (500, 501), (503, 1001)), want):
        assert (np.abs(got[lo:hi] - w) <= np.abs(w) * 3 * 2.0 ** -24).all()
    m = rng.randn(40, 60).astype(np.float32)
    t = D.Array.from_numpy(m)
    got, _ = D.op.clip_by_global_norm([t.T, t[:, 5:9], t * 2.0], 1.0)
    want, _ = reference([m.T, m[:, 5:9], m * 2], 1.0)
    assert all((np.abs(g.numpy() - w) <= np.abs(w) * 3 * 2.0 ** -24).all() for g, w in zip(got, want))


def test_results_that_repeat(gpu, D, rng):
    held = [D.Array.from_numpy(rng.randn(n).astype(np.float32)) for n in (1 << 21, 1000, 77777)]
    want, norm = D.op.clip_by_global_norm(held, 1.0)
    for _ in range(5):
        got, again = D.op.clip_by_global_norm(held, 1.0)
        assert np.array_equal(norm.numpy(), again.numpy()) and all(np.array_equal(p.numpy(), q.numpy()) for p, q in zip(got, want))


def test_recorded(gpu, D, rng):
    for n in (500, 300000):
        x = D.Array.from_numpy(rng.randn(n).astype(np.float32))
        fill = [D.Array.empty((n,)), D.Array.from_numpy(rng.randn(9).astype(np.float32))]
        fill[0].assign(x)
        with D.Recording() as rec:
            got, norm = D.op.clip_by_global_norm(fill, 3.0)
        for graph in (False, True):
            if graph:
                rec.make_graph()
            for step in range(3):
                fill[0].assign(x * float(step + 1))
                rec.replay()
                want, again = D.op.clip_by_global_norm(fill, 3.0)
                assert np.array_equal(norm.numpy(), again.numpy()) and all(np.array_equal(p.numpy(), q.numpy()) for p, q in zip(got, want)), (graph, step)


def test_device_refusals(gpu, D, rng):
    op = D.op
    buf = D.Array.from_numpy(rng.randn(100).astype(np.float32))
    before = buf.numpy()
    a, b = buf[0:40], buf[40:80]
    with pytest.raises(D.DaliError, match="result 0 overlaps array 1"):
        op.clip_by_global_norm([a, b], 1.0, out=([b, None], None))
    with pytest.raises(D.DaliError, match="results 0 and 1 overlap"):
        op.clip_by_global_norm([a, a], 1.0, out=([b, b], None))
    with pytest.raises(D.DaliError, match="results 0 and 1 overlap"):
        op.clip_by_global_norm([a, a], 1.0, out=([a, a], None))
    with pytest.raises(D.DaliError, match="result 0 overlaps array 0"):
        op.clip_by_global_norm([a], 1.0, out=([buf[1:41]], None))
    with pytest.raises(D.DaliError, match="result 1 overlaps array 0"):
        op.clip_by_global_norm([buf[0:60], buf[10:60]], 1.0, out=([None, buf[10:60]], None))
    with pytest.raises(D.DaliError, match="norm overlaps"):
        op.clip_by_global_norm([a], 1.0, out=(None, buf[3]))
    assert np.array_equal(buf.numpy(), before)

"""Layer normalisation and its gradient against the formulas in higher precision: widths and row counts around every change of the kernels, views, destinations.

u is half a unit in the last place of 1. A sum of n terms in the kernels is at most n / 64 additions deep for one thread, some more over a wave and a workgroup:
`depth` below; its error is at most depth * u * the sum of the magnitudes.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = {np.float32: 2.0 ** -24, np.float64: 2.0 ** -53}
# one thread and less than a wave of values, around a wave, around the whole 16-byte pieces of a wave, two waves ... and rows that no workgroup holds
WIDTHS = [1, 2, 3, 5, 16, 31, 63, 64, 65, 97, 128, 255, 256, 257, 260, 511, 512, 513, 768, 1000, 1023, 1024, 1025, 1536, 2047, 2048, 2049, 4095, 4096, 4100, 8192, 8193,
          16384, 16388, 32769]


def depth(n):
    return n / 64 + 32


def oracle(x, gamma, beta, epsilon):
    x, gamma, beta = (v.astype(np.longdouble) for v in (x, gamma, beta))
    mean = x.mean(-1)
    d = x - mean[..., None]
    rstd = 1 / np.sqrt((d * d).mean(-1) + epsilon)
    return d * rstd[..., None] * gamma + beta, mean, rstd


def check_forward(x, gamma, beta, epsilon, got):
    u = U[x.dtype.type]
    y, mean, rstd = got
    want, wmean, wrstd = oracle(x, gamma, beta, epsilon)
    n = x.shape[-1]
    tol = (depth(n) + 16) * u
    spread = np.abs(x - wmean[..., None]).mean(-1)
    assert (np.abs(mean - wmean) <= u * np.abs(wmean) + tol * spread + tol * u * np.abs(x).mean(-1)).all()
    # (the mean as it is subtracted is off by tol of the spread, and by tol^2 of the values' own size)
    lost = (tol * tol * np.abs(x).mean(-1) + tol * spread) * wrstd
    assert (np.abs(rstd - wrstd) <= wrstd * (tol + lost * lost)).all()
    unit = np.abs((want - beta) / np.where(gamma == 0, 1, gamma))
    assert (np.abs(y - want) <= np.abs(gamma) * (lost[..., None] + (tol + (lost * lost)[..., None]) * unit) + 2 * u * (np.abs(beta) + np.abs(want))).all()


def case(rng, rows, width, dtype, shift=0, offset=0.3):
    full = (rng.randn(rows, width + shift) * 2 + offset).astype(dtype)
    gamma, beta = (1 + 0.2 * rng.randn(width)).astype(dtype), (0.2 * rng.randn(width)).astype(dtype)
    return full, full[:, shift:], gamma, beta


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_forward(gpu, D, rng, width, dtype):
    for rows, shift in ((1, 0), (3, 1), (70, 0), (513 if width <= 4100 else 17, 3)):
        full, x, gamma, beta = case(rng, rows, width, dtype, shift)
        a = D.Array.from_numpy(full)
        a = a[:, shift:] if shift else a
        got = D.op.layer_norm(a, D.Array.from_numpy(gamma), D.Array.from_numpy(beta), 1e-5)
        assert [v.shape for v in got] == [(rows, width), (rows,), (rows,)]
        check_forward(x, gamma, beta, 1e-5, [v.numpy() for v in got])


def backward_bounds(dy, x, mean, rstd, gamma):
    u = U[x.dtype.type]
    dy, x, mean, rstd, gamma = (v.astype(np.longdouble) for v in (dy, x, mean, rstd, gamma))
    n, rows = x.shape[-1], x.shape[0]
    unit = (x - mean[:, None]) * rstd[:, None]
    a = dy * gamma
    level, along = a.mean(1)[:, None], (a * unit).mean(1)[:, None]
    dx = rstd[:, None] * (a - level - unit * along)
    tol = (depth(n) + 16) * u
    dx_bound = rstd[:, None] * (tol * (np.abs(a).mean(1)[:, None] + np.abs(unit) * np.abs(a * unit).mean(1)[:, None]) + 8 * u * (np.abs(a) + np.abs(level) + np.abs(unit * along)))
    # over the rows: at least 32 parts of them, each summed on its own, then the parts
    down = (rows / 32 + 1024 + 8) * u
    return (dx, dx_bound), ((dy * unit).sum(0), down * np.abs(dy * unit).sum(0)), (dy.sum(0), down * np.abs(dy).sum(0))


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_backward(gpu, D, rng, width, dtype):
    for rows, shift in ((1, 0), (3, 1), (70, 0), (1030 if width <= 4100 else 17, 3)):
        full, x, gamma, beta = case(rng, rows, width, dtype, shift)
        _, mean, rstd = oracle(x, gamma, beta, 1e-5)
        mean, rstd = mean.astype(dtype), rstd.astype(dtype)
        dy = rng.randn(rows, width).astype(dtype)
        a = D.Array.from_numpy(full)
        a = a[:, shift:] if shift else a
        got = D.op.layer_norm_backward(*[D.Array.from_numpy(dy), a] + [D.Array.from_numpy(v) for v in (mean, rstd, gamma)])
        for g, (want, bound) in zip(got, backward_bounds(dy, x, mean, rstd, gamma)):
            assert g.shape == want.shape
            assert (np.abs(g.numpy() - want) <= bound + 1e-300).all(), (rows, shift)


@pytest.mark.parametrize("rows", [1, 2, 31, 32, 33, 255, 256, 257, 1000, 4099, 20011])
@pytest.mark.parametrize("width", [1, 7, 64, 96, 200, 1028])
def test_gradients_of_the_weights_miss_no_row(gpu, D, rows, width):
    """Whole numbers: every sum is exact, in any order."""
    rng = np.random.RandomState(rows + width)
    x, dy = rng.randint(-8, 9, (rows, width)).astype(np.float32), rng.randint(-8, 9, (rows, width)).astype(np.float32)
    mean, rstd = rng.randint(-2, 3, rows).astype(np.float32), np.exp2(rng.randint(-1, 2, rows)).astype(np.float32)
    dx, dgamma, dbeta = D.op.layer_norm_backward(*[D.Array.from_numpy(v) for v in (dy, x, mean, rstd, np.ones(width, np.float32))])
    unit = (x - mean[:, None]) * rstd[:, None]
    assert np.array_equal(dgamma.numpy(), (dy * unit).astype(np.float64).sum(0))
    assert np.array_equal(dbeta.numpy(), dy.astype(np.float64).sum(0))


@pytest.mark.parametrize("width", [5, 96, 300, 1024, 5000])
def test_gradient_against_differences(gpu, D, rng, width):
    rows, step = 3, 1e-6
    _, x, gamma, beta = case(rng, rows, width, np.float64)
    dy = rng.randn(rows, width)

    def loss(x, gamma, beta):
        return float((D.op.layer_norm(*[D.Array.from_numpy(v) for v in (x, gamma, beta)])[0].numpy() * dy).sum())

    _, mean, rstd = D.op.layer_norm(*[D.Array.from_numpy(v) for v in (x, gamma, beta)])
    grads = [g.numpy() for g in D.op.layer_norm_backward(D.Array.from_numpy(dy), D.Array.from_numpy(x), mean, rstd, D.Array.from_numpy(gamma))]
    for which, grad in enumerate(grads):
        along = rng.randn(*grad.shape)
        ends = []
        for sign in (1, -1):
            moved = [x, gamma, beta]
            moved[which] = moved[which] + sign * step * along
            ends.append(loss(*moved))
        # the slope along a direction: third derivatives are of the size of the loss's terms (step^2), rounding of the loss over the step
        scale = np.abs(dy).sum() * 10
        assert abs((ends[0] - ends[1]) / (2 * step) - (grad * along).sum()) <= scale * (100 * step ** 2 + 1e-16 * 100 / step)


@pytest.mark.parametrize("width", [1, 64, 1000, 4096, 20000])
def test_rows_without_spread_and_far_from_zero(gpu, D, rng, width):
    constant = np.full((4, width), 3.25, np.float32)
    constant[1] = 0
    constant[2] = -1e30
    y, mean, rstd = (v.numpy() for v in D.op.layer_norm(D.Array.from_numpy(constant)))
    assert np.array_equal(y[:2], np.zeros((2, width), np.float32)) and np.array_equal(mean[:2], constant[:2, 0])
    np.testing.assert_allclose(rstd[:2], 1e-5 ** -0.5, rtol=4 * 2.0 ** -24)
    assert np.array_equal(y[3], np.zeros(width, np.float32))
    far = (rng.randn(6, width) + 10000.0).astype(np.float32)
    got = [v.numpy() for v in D.op.layer_norm(D.Array.from_numpy(far))]
    check_forward(far, np.ones(width, np.float32), np.zeros(width, np.float32), 1e-5, got)


@pytest.mark.parametrize("width", [3, 100, 1024, 1030, 9000])
def test_infinities_and_nan_stay_in_their_rows(gpu, D, rng, width):
    x = rng.randn(9, width).astype(np.float32)
    x[1, 0], x[4, width - 1], x[7, width // 2] = np.nan, np.inf, -np.inf
    y, mean, rstd = (v.numpy() for v in D.op.layer_norm(D.Array.from_numpy(x)))
    bad = [1, 4, 7]
    assert np.isnan(y[bad]).any(1).all()
    good = [0, 2, 3, 5, 6, 8]
    check_forward(x[good], np.ones(width, np.float32), np.zeros(width, np.float32), 1e-5, [y[good], mean[good], rstd[good]])


def test_shapes_views_and_absent_weights(gpu, D, rng):
    x = rng.randn(4, 6, 8, 96).astype(np.float32)
    a = D.Array.from_numpy(x)
    one, zero = np.ones(96, np.float32), np.zeros(96, np.float32)
    views = [(a, x), (a[:, 2], x[:, 2]), (a[1:3, ::2], x[1:3, ::2]), (a[:, :, ::-1], x[:, :, ::-1]), (a.transpose(2, 0, 1, 3), x.transpose(2, 0, 1, 3)),
             (a.transpose(0, 3, 2, 1), x.transpose(0, 3, 2, 1)), (a[:, :, :, 1:], x[..., 1:]), (a[0, 0, 0], x[0, 0, 0])]
    for view, ref in views:
        n = ref.shape[-1]
        y, mean, rstd = D.op.layer_norm(view)
        assert y.shape == ref.shape and mean.shape == ref.shape[:-1] == rstd.shape
        check_forward(np.ascontiguousarray(ref), np.ones(n, np.float32), np.zeros(n, np.float32), 1e-5, [v.numpy() for v in (y, mean, rstd)])
        dy = rng.randn(*ref.shape).astype(np.float32)
        dx, dgamma, dbeta = D.op.layer_norm_backward(D.Array.from_numpy(dy), view, mean, rstd)
        assert dgamma is None and dbeta is None
        flat = [np.ascontiguousarray(v).reshape(-1, n) for v in (dy, ref)] + [v.numpy().reshape(-1) for v in (mean, rstd)]
        want, bound = backward_bounds(*flat, np.ones(n, np.float32))[0]
        assert (np.abs(dx.numpy().reshape(-1, n) - want) <= bound).all()
    # a lazily built operand, and only one of the weights
    gamma = (1 + rng.randn(96)).astype(np.float32)
    y = D.op.layer_norm(a * 2.0, gamma=D.Array.from_numpy(gamma))[0].numpy()
    assert (np.abs(y - oracle(x * 2, gamma, zero, 1e-5)[0]) <= 1e-4).all()
    y = D.op.layer_norm(a, beta=D.Array.from_numpy(gamma))[0].numpy()
    assert (np.abs(y - oracle(x, one, gamma, 1e-5)[0]) <= 1e-4).all()


@pytest.mark.parametrize("rows,width", [(0, 7), (5, 64), (300, 1024), (40, 5000), (7, 40000)])
def test_destinations(gpu, D, rng, rows, width):
    op = D.op
    x, dy = rng.randn(rows, width).astype(np.float32), rng.randn(rows, width).astype(np.float32)
    gamma = D.Array.from_numpy((1 + rng.randn(width)).astype(np.float32))
    y, mean, rstd = op.layer_norm(D.Array.from_numpy(x), gamma)
    dx, dgamma, dbeta = op.layer_norm_backward(D.Array.from_numpy(dy), D.Array.from_numpy(x), mean, rstd, gamma)
    if rows == 0:
        assert y.numpy().shape == (0, 7) and not dgamma.numpy().any() and not dbeta.numpy().any()
    # in the operand's place, beside it, and inside a larger buffer whose other values stay
    a = D.Array.from_numpy(x)
    got = op.layer_norm(a, gamma, out=(a, None, None))
    assert got[0] is a and np.array_equal(a.numpy(), y.numpy()) and np.array_equal(got[1].numpy(), mean.numpy())
    for place in (0, 1):
        b = [D.Array.from_numpy(dy), D.Array.from_numpy(x)]
        got = op.layer_norm_backward(b[0], b[1], mean, rstd, gamma, out=(b[place], None, None))
        assert np.array_equal(b[place].numpy(), dx.numpy()) and np.array_equal(got[1].numpy(), dgamma.numpy()) and np.array_equal(got[2].numpy(), dbeta.numpy())
    big = D.Array.from_numpy(np.full((rows + 2, width), 7, np.float32))
    op.layer_norm(D.Array.from_numpy(x), gamma, out=(big[1:rows + 1], None, None))
    assert np.array_equal(big.numpy()[1:-1], y.numpy()) and (big.numpy()[[0, -1]] == 7).all()


def test_a_row_apart_and_results_that_repeat(gpu, D, rng):
    """A row's result does not depend on the others, nor any result on the run."""
    x, dy = rng.randn(3000, 1024).astype(np.float32), rng.randn(3000, 1024).astype(np.float32)
    a, g = D.Array.from_numpy(x), D.Array.from_numpy(dy)
    gamma = D.Array.from_numpy((1 + rng.randn(1024)).astype(np.float32))
    first = D.op.layer_norm(a, gamma)
    grads = D.op.layer_norm_backward(g, a, first[1], first[2], gamma)
    for _ in range(3):
        assert all(np.array_equal(p.numpy(), q.numpy()) for p, q in zip(first, D.op.layer_norm(a, gamma)))
        assert all(np.array_equal(p.numpy(), q.numpy()) for p, q in zip(grads, D.op.layer_norm_backward(g, a, first[1], first[2], gamma)))


def test_recorded(gpu, D, rng):
    op = D.op
    x, gamma = D.Array.from_numpy(rng.randn(50, 300).astype(np.float32)), D.Array.from_numpy(rng.randn(300).astype(np.float32))
    fill = D.Array.empty((50, 300))
    fill.assign(x)
    with D.Recording() as rec:
        y, mean, rstd = op.layer_norm(fill, gamma)
        dx, dgamma, dbeta = op.layer_norm_backward(y, fill, mean, rstd, gamma)
    rec.replay()
    for graph in (False, True):
        if graph:
            rec.make_graph()
        for step in range(3):
            fill.assign(x * float(step + 2))
            rec.replay()
            want = op.layer_norm(fill, gamma)
            back = op.layer_norm_backward(want[0], fill, want[1], want[2], gamma)
            for p, q in zip((y, mean, rstd, dx, dgamma, dbeta), want + back):
                assert np.array_equal(p.numpy(), q.numpy()), (graph, step)


def test_device_refusals(gpu, D, rng):
    op = D.op
    buf = D.Array.from_numpy(rng.randn(64, 64).astype(np.float32))
    before = buf.numpy()
    small = buf[:8]
    with pytest.raises(D.DaliError, match="y overlaps x"):
        op.layer_norm(buf[0:8], out=(buf[4:12], None, None))
    with pytest.raises(D.DaliError, match="mean overlaps x"):
        op.layer_norm(small, out=(None, buf[0, :8], None))
    with pytest.raises(D.DaliError, match="y and mean overlap"):
        op.layer_norm(D.Array.from_numpy(before[:8]), out=(buf[:8], buf[1, :8], None))
    with pytest.raises(D.DaliError, match="overlaps x"):
        op.layer_norm(buf[:8, :32], out=(buf[:4].reshape(8, 32), None, None))
    stats = [D.Array.from_numpy(np.ones(8, np.float32)) for _ in range(2)]
    with pytest.raises(D.DaliError, match="dx overlaps dy"):
        op.layer_norm_backward(buf[0:8], D.Array.from_numpy(before[:8]), *stats, out=(buf[1:9], None, None))
    for epsilon in (-1.0, float("nan")):
        with pytest.raises(D.DaliError, match="epsilon"):
            op.layer_norm(small, epsilon=epsilon)
    assert np.array_equal(buf.numpy(), before)

"""Attention to an encoder's states and its gradients against the formulas in 64 bits: lengths around every change of the kernels, shared heads, padded batches, views.

u is half a unit in the last place of 1. A score is a sum of `width` products of a factor that is rounded twice: off by at most (width + 4) u of the sum A of the products'
magnitudes (times the scale). A weight e^(s - m) is then off by twice that (its maximum is a score too), by the rounding of s - m, and by 4 u for the exponential: `weight`
below, relative. A result is a sum over n weights, with at most as many rescalings as states: 2 (n + 8) u more of the sum of the magnitudes, and the sum that it is
divided by as much again.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = {np.float32: 2.0 ** -24, np.float64: 2.0 ** -53}


def heads_of(x, group):
    """[batch, positions, kv heads, width] -> [batch, heads, positions, width] in 64 bits or more"""
    wide = np.longdouble if x.dtype == np.float64 else np.float64
    return np.repeat(x.astype(wide), group, axis=2).transpose(0, 2, 1, 3)


def scores(q, k, counts, scale):
    qh, kh = heads_of(q, 1), heads_of(k, q.shape[2] // k.shape[2])
    turned = np.ascontiguousarray(kh.transpose(0, 1, 3, 2))
    there = np.arange(k.shape[1])[None, :] < counts[:, None]
    s = np.where(there[:, None, None, :], np.matmul(qh, turned) * scale, -np.inf)
    size = np.where(there[:, None, None, :], np.matmul(np.abs(qh), np.abs(turned)) * abs(scale), 0)
    return s, size


def forward(q, k, v, counts, scale):
    u = U[q.dtype.type]
    n = np.clip(counts, 0, k.shape[1])
    v = np.where((np.arange(k.shape[1])[None, :] < n[:, None])[:, :, None, None], v, 0)
    k = np.where((np.arange(k.shape[1])[None, :] < n[:, None])[:, :, None, None], k, 0)
    s, size = scores(q, k, n, scale)
    if k.shape[1] == 0:
        s, size = np.full(s.shape[:3] + (1,), -np.inf), np.zeros(size.shape[:3] + (1,))
        v = np.zeros((v.shape[0], 1) + v.shape[2:], v.dtype)
    top = s.max(-1, keepdims=True)
    top = np.where(np.isfinite(top), top, 0)
    w = np.exp(s - top)
    total = w.sum(-1, keepdims=True)
    with np.errstate(divide="ignore"):
        lse = (top + np.log(total))[..., 0]
    p = w / np.where(total == 0, 1, total)
    vh = heads_of(v, q.shape[2] // v.shape[2])
    y = np.matmul(p, vh)
    spread = np.where(np.isfinite(s), np.abs(s - top), 0).max(-1)
    weight = 2 * (q.shape[3] + 4) * u * size.max(-1) + u * (spread + 4)
    sums = 2 * (s.shape[-1] + 8) * u
    y_bound = (2 * weight + 2 * sums)[..., None] * np.matmul(p, np.abs(vh))
    lse_bound = weight + sums + 4 * u * np.abs(np.where(np.isfinite(lse), lse, 0)) + 4 * u * np.abs(top[..., 0])
    back = lambda x: np.moveaxis(x, 1, 2)  # noqa: E731
    return back(y), back(lse), back(y_bound), back(lse_bound)


def make(rng, dtype, batch, queries, keys, heads, kv_heads, width, counts=None):
    q, k, v = (rng.randn(batch, n, h, width).astype(dtype) for n, h in ((queries, heads), (keys, kv_heads), (keys, kv_heads)))
    if counts is None:
        counts = rng.randint(0, keys + 1, batch)
        counts[rng.randint(batch)] = keys
    counts = np.asarray(counts, np.int32)
    return q, k, v, counts


def near(got, want, bound):
    empty = ~np.isfinite(want)
    assert np.array_equal(got[empty], want[empty])
    off = np.abs(got[~empty] - want[~empty])
    assert (off <= bound[~empty]).all(), (off / np.maximum(bound[~empty], 1e-300)).max()


def check_forward(D, q, k, v, counts, scale, got=None):
    A = D.Array.from_numpy
    y, lse = got or D.op.cross_attention(A(q), A(k), A(v), A(counts), scale)
    assert y.shape == q.shape and lse.shape == q.shape[:3]
    wy, wl, by, bl = forward(q, k, v, counts, scale)
    near(lse.numpy(), wl, bl)
    near(y.numpy(), wy, by)
    return y, lse


SIZES = [(1, 1, 1, 1, 1, 1), (1, 1, 5, 2, 2, 3), (3, 1, 17, 4, 1, 16), (2, 1, 300, 16, 2, 64), (2, 2, 64, 8, 8, 64), (1, 1, 65, 1, 1, 128), (5, 4, 33, 5, 5, 40),
         (2, 16, 31, 1, 1, 32), (2, 17, 129, 1, 1, 33), (1, 32, 200, 2, 2, 64), (1, 33, 63, 2, 1, 64), (3, 37, 95, 6, 3, 48), (2, 64, 64, 2, 2, 31), (2, 65, 257, 4, 2, 65),
         (1, 130, 97, 3, 3, 128), (2, 129, 161, 2, 2, 100), (1, 70, 70, 2, 1, 129), (2, 35, 67, 2, 2, 200), (1, 40, 50, 2, 2, 256), (1, 3, 90, 3, 3, 256), (1, 20, 90, 1, 1, 255),
         (1, 257, 1000, 1, 1, 64), (2, 1, 4097, 3, 1, 80), (1, 40, 2000, 2, 2, 16), (70, 3, 9, 8, 4, 8)]


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_forward(gpu, D, rng, size, dtype):
    q, k, v, counts = make(rng, dtype, *size)
    check_forward(D, q, k, v, counts, 1 / np.sqrt(size[5]))


def backward(dy, q, k, v, y, lse, counts, scale):
    u, (batch, queries, heads, width), group, states = U[q.dtype.type], q.shape, q.shape[2] // k.shape[2], k.shape[1]
    n = np.clip(counts, 0, states)
    there = (np.arange(states)[None, :] < n[:, None])[:, :, None, None]
    k, v = np.where(there, k, 0), np.where(there, v, 0)
    s, size = scores(q, k, n, scale)
    qh, gh, yh = heads_of(q, 1), heads_of(dy, 1), heads_of(y, 1)
    kh, vh = heads_of(k, group), heads_of(v, group)
    level = lse.astype(qh.dtype).transpose(0, 2, 1)[..., None]
    p = np.where(np.isfinite(s) & np.isfinite(level), np.exp(np.where(np.isfinite(s), s, 0) - np.where(np.isfinite(level), level, 0)), 0)
    T = lambda x: np.ascontiguousarray(x.transpose(0, 1, 3, 2))  # noqa: E731
    dp, dp_size = np.matmul(gh, T(vh)), np.matmul(np.abs(gh), T(np.abs(vh)))
    delta, delta_size = (gh * yh).sum(-1, keepdims=True), np.abs(gh * yh).sum(-1, keepdims=True)
    ds = p * (dp - delta)
    exponents = np.where(np.isfinite(s), np.abs(s), 0) + np.where(np.isfinite(level), np.abs(level), 0)
    p_bound = p * (2 * (width + 4) * u * size + 2 * u * exponents + 6 * u)
    ds_bound = p_bound * np.abs(dp - delta) + p * (width + 6) * u * (dp_size + delta_size)
    rows = queries * group
    dq, dq_bound = np.matmul(ds, kh) * scale, np.matmul(ds_bound + (states + 4) * u * np.abs(ds), np.abs(kh)) * abs(scale)
    dk, dk_bound = np.matmul(T(ds), qh) * scale, np.matmul(T(ds_bound + (rows + 4) * u * np.abs(ds)), np.abs(qh)) * abs(scale)
    dv, dv_bound = np.matmul(T(p), gh), np.matmul(T(p_bound + (rows + 4) * u * p), np.abs(gh))
    fold = lambda x: x.reshape(batch, heads // group, group, states, width).sum(2).transpose(0, 2, 1, 3)  # noqa: E731
    back = lambda x: x.transpose(0, 2, 1, 3)  # noqa: E731
    return (back(dq), back(dq_bound)), (fold(dk), fold(dk_bound)), (fold(dv), fold(dv_bound))


def check_backward(D, dy, q, k, v, counts, scale, got=None):
    A = D.Array.from_numpy
    y, lse = D.op.cross_attention(A(q), A(k), A(v), A(counts), scale)
    got = got or D.op.cross_attention_backward(A(dy), A(q), A(k), A(v), y, lse, A(counts), scale)
    for g, (want, bound), shape in zip(got, backward(dy, q, k, v, y.numpy(), lse.numpy(), counts, scale), (q.shape, k.shape, k.shape)):
        assert g.shape == shape
        near(g.numpy(), want, bound)
    behind = np.arange(k.shape[1])[None, :] >= counts[:, None]
    assert (got[1].numpy()[behind] == 0).all() and (got[2].numpy()[behind] == 0).all()
    return got


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_backward(gpu, D, rng, size, dtype):
    q, k, v, counts = make(rng, dtype, *size)
    check_backward(D, rng.randn(*q.shape).astype(dtype), q, k, v, counts, 1 / np.sqrt(size[5]))


@pytest.mark.parametrize("queries", [1, 20, 70])
@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_what_lies_behind_the_last_state_is_not_read(gpu, D, rng, queries, dtype):
    keys = 150
    for bad in (np.nan, np.inf, -np.inf, np.finfo(dtype).max, np.finfo(dtype).min):
        q, k, v, counts = make(rng, dtype, 6, queries, keys, 4, 2, 24, [0, 1, 63, 64, 149, 150])
        behind = np.arange(keys)[None, :] >= counts[:, None]
        clean = D.op.cross_attention(*(D.Array.from_numpy(a) for a in (q, k, v, counts)))
        k[behind], v[behind] = bad, bad
        check_forward(D, q, k, v, counts, 1 / np.sqrt(24))
        dirty = D.op.cross_attention(*(D.Array.from_numpy(a) for a in (q, k, v, counts)))
        assert all(np.array_equal(a.numpy(), b.numpy()) for a, b in zip(clean, dirty))
        check_backward(D, rng.randn(*q.shape).astype(dtype), q, k, v, counts, 1 / np.sqrt(24))


def test_counts_are_held_inside(gpu, D, rng):
    q, k, v, _ = make(rng, np.float32, 4, 5, 40, 2, 2, 16)
    for queries in (5, 40):
        q = rng.randn(4, queries, 2, 16).astype(np.float32)
        wild = np.array([-1, 41, np.iinfo(np.int32).max, np.iinfo(np.int32).min], np.int32)
        check_forward(D, q, k, v, wild, 0.25)
        check_backward(D, rng.randn(*q.shape).astype(np.float32), q, k, v, np.clip(wild, 0, 40), 0.25)
        A = D.Array.from_numpy
        for a, b in zip(D.op.cross_attention(A(q), A(k), A(v)), D.op.cross_attention(A(q), A(k), A(v), A(np.full(4, 40, np.int32)), 0.25)):
            assert np.array_equal(a.numpy(), b.numpy())


@pytest.mark.parametrize("queries", [2, 50])
def test_no_states_and_no_positions(gpu, D, rng, queries):
    A = D.Array.from_numpy
    q, k = rng.randn(2, queries, 3, 8).astype(np.float32), np.zeros((2, 0, 3, 8), np.float32)
    y, lse = D.op.cross_attention(A(q), D.Array.empty(k.shape), D.Array.empty(k.shape))
    assert (y.numpy() == 0).all() and (lse.numpy() == -np.inf).all()
    dq, dk, dv = D.op.cross_attention_backward(A(q), A(q), D.Array.empty(k.shape), D.Array.empty(k.shape), y, lse)
    assert (dq.numpy() == 0).all() and dk.shape == dv.shape == k.shape
    k = rng.randn(2, 70, 3, 8).astype(np.float32)
    none = D.Array.empty((2, 0, 3, 8))
    y, lse = D.op.cross_attention(none, A(k), A(k))
    assert y.shape == (2, 0, 3, 8) and lse.shape == (2, 0, 3)
    dq, dk, dv = D.op.cross_attention_backward(none, none, A(k), A(k), y, lse)
    assert (dk.numpy() == 0).all() and (dv.numpy() == 0).all()


@pytest.mark.parametrize("queries", [1, 3, 60])
@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_large_and_infinite_scores(gpu, D, rng, queries, dtype):
    """Scores far from 0, a row whose scores are all -inf, one with a NaN: each stays with its row."""
    q, k, v, counts = make(rng, dtype, 2, queries, 130, 2, 2, 16, [130, 77])
    check_forward(D, q * 30, k, v, counts, 0.5)
    check_backward(D, rng.randn(*q.shape).astype(dtype), q * 8, k, v, counts, 0.5)
    check_forward(D, q, k, v, counts, -0.25)
    check_forward(D, q, k, v, counts, 0.0)
    k[0, :, 0, 0], q[0, :, :, 0] = -np.inf, np.abs(q[0, :, :, 0]) + 1
    q[0, -1, 1] = np.nan
    A = D.Array.from_numpy
    y, lse = D.op.cross_attention(A(q), A(k), A(v), A(counts), 0.25)
    y, lse = y.numpy(), lse.numpy()
    assert (y[0, :-1, 0] == 0).all() and (lse[0, :, 0] == -np.inf).all()
    assert np.isnan(y[0, -1, 1]).all() and np.isnan(lse[0, -1, 1])
    assert np.isfinite(y[1]).all() and np.isfinite(y[0, :-1, 1]).all()
    q[0, -1, 1] = 0
    d = D.op.cross_attention_backward(A(q), A(q), A(k), A(v), A(np.where(np.isnan(y), 0, y)), A(np.where(np.isnan(lse), 0, lse)), A(counts), 0.25)
    assert np.isfinite(d[2].numpy()).all() and (d[2].numpy()[0, :, 0] == 0).all()  # (rows without weight give the values nothing)


@pytest.mark.parametrize("queries", [1, 70])
@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_views_and_destinations(gpu, D, rng, queries, dtype):
    A, op, scale = D.Array.from_numpy, D.op, 0.2
    q, k, v, counts = make(rng, dtype, 3, queries, 90, 4, 2, 24, [90, 0, 33])
    dy = rng.randn(*q.shape).astype(dtype)
    turned = lambda a: A(np.ascontiguousarray(a.transpose(0, 2, 1, 3))).transpose(0, 2, 1, 3)  # noqa: E731
    plain = op.cross_attention(A(q), A(k), A(v), A(counts), scale)
    grads = check_backward(D, dy, q, k, v, counts, scale)
    # [batch, heads, positions, width]; keys and values side by side in one array; every other state of a longer one; a last axis that is not dense
    both = A(np.concatenate([k, v], 2))
    longer = A(np.repeat(k, 2, 1))
    for views in ((turned(q), turned(k), turned(v)), (A(q), both[:, :, :2], both[:, :, 2:]), (A(q), longer[:, ::2], A(v)),
                  (A(np.ascontiguousarray(q.transpose(3, 0, 1, 2))).transpose(1, 2, 3, 0), A(k), A(v)), (A(q[:, ::-1].copy())[:, ::-1], A(k), A(v))):
        for a, b in zip(plain, op.cross_attention(*views, A(counts), scale)):
            assert np.array_equal(a.numpy(), b.numpy())
        for a, b in zip(grads, op.cross_attention_backward(turned(dy), *views, *plain, A(counts), scale)):
            assert np.array_equal(a.numpy(), b.numpy())
    outs = tuple(A(np.full(s, np.nan, dtype)) for s in (q.shape, q.shape[:3]))
    assert all(a is b for a, b in zip(op.cross_attention(A(q), A(k), A(v), A(counts), scale, out=outs), outs))
    check_forward(D, q, k, v, counts, scale, outs)
    outs = tuple(A(np.full(s, np.nan, dtype)) for s in (q.shape, k.shape, k.shape))
    op.cross_attention_backward(A(dy), A(q), A(k), A(v), *plain, A(counts), scale, out=outs)
    assert all(np.array_equal(a.numpy(), b.numpy()) for a, b in zip(grads, outs))
    # keys that are the values, lazily built operands
    check_forward(D, q, k, k, counts, scale, op.cross_attention(A(q) * 1.0, *[A(k)] * 2, A(counts), scale))


def test_gradients_against_differences(gpu, D, rng):
    """d(sum y c)/dx by central differences in double: the error of a step h is h^2 / 6 of a third derivative of order 1 and u / h of rounding: below 1e-7 at h = 1e-4."""
    A, op = D.Array.from_numpy, D.op
    q, k, v, counts = make(rng, np.float64, 2, 3, 7, 4, 2, 5, [7, 4])
    c = rng.randn(*q.shape)
    y, lse = op.cross_attention(A(q), A(k), A(v), A(counts), 0.4)
    grads = op.cross_attention_backward(A(c), A(q), A(k), A(v), y, lse, A(counts), 0.4)
    for which, g in enumerate(grads):
        for _ in range(12):
            at = tuple(rng.randint(n) for n in (q, k, v)[which].shape)
            value = []
            for h in (1e-4, -1e-4):
                moved = [q.copy(), k.copy(), v.copy()]
                moved[which][at] += h
                value.append((op.cross_attention(*(A(m) for m in moved), A(counts), 0.4)[0].numpy() * c).sum())
            assert abs((value[0] - value[1]) / 2e-4 - g.numpy()[at]) < 1e-6


@pytest.mark.parametrize("queries", [1, 24, 100])
def test_recorded_and_replayed(gpu, D, rng, queries):
    A, op = D.Array.from_numpy, D.op
    q, k, v, counts = make(rng, np.float32, 2, queries, 700, 4, 4, 32, [700, 123])
    dy = rng.randn(*q.shape).astype(np.float32)
    qa, ka, va, ga, na = A(q), A(k), A(v), A(dy), A(counts)
    outs = [D.Array.empty(s) for s in (q.shape, q.shape[:3], q.shape, k.shape, k.shape)]
    rec, other = D.Recording(), D.Recording()
    for r in (rec, other):  # (two recordings of the same call do not share what they keep)
        with r:
            op.cross_attention(qa, ka, va, na, 0.2, out=outs[:2])
            op.cross_attention_backward(ga, qa, ka, va, outs[0], outs[1], na, 0.2, out=outs[2:])
        r.make_graph()
    for step in range(3):
        qa.assign(qa * -0.7)
        na.assign(A(np.array([step * 300, 699], np.int32)))
        for o in outs:
            o.assign(o * 0.0)
        op.cross_attention(qa * 2.0, ka, va)[0].numpy()  # the program's own work in between
        rec.replay()
        other.replay()
        check_forward(D, qa.numpy(), k, v, na.numpy(), 0.2, outs[:2])
        check_backward(D, dy, qa.numpy(), k, v, na.numpy(), 0.2, outs[2:])

"""Embedding rows and the gradient of the table against the formulas in 64 bits and more: widths and counts around every change of the kernels, tokens outside, heavy tokens, views.

u is half a unit in the last place of 1. A row is one product: off by u of its value at most. A row of the gradient is the sum of n rows of dy and one product: n + 1 roundings, each
of at most the sum of the magnitudes.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = {np.float32: 2.0 ** -24, np.float64: 2.0 ** -53}
WIDTHS = [1, 2, 3, 4, 5, 7, 8, 31, 32, 33, 63, 64, 97, 127, 128, 129, 130, 255, 256, 257, 511, 513, 1024, 1027, 2049, 4100]


def tokens_of(rng, count, rows, outside=True):
    t = np.minimum((rows ** rng.rand(count)).astype(np.int64) - 1, rows - 1).astype(np.int32)
    if outside and count > 3:
        t[rng.randint(0, count, max(1, count // 9))] = -1
        t[rng.randint(0, count)] = rows
        t[rng.randint(0, count)] = np.iinfo(np.int32).max
        t[rng.randint(0, count)] = np.iinfo(np.int32).min
    return t


def check_rows(y, table, tokens, scale):
    inside = (tokens >= 0) & (tokens < table.shape[0])
    want = np.where(inside[:, None], table.astype(np.longdouble)[np.where(inside, tokens, 0)] * np.longdouble(scale), 0)
    assert (np.abs(y - want) <= U[table.dtype.type] * np.abs(want)).all()


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_rows(gpu, D, rng, width, dtype):
    for count, rows, shift in ((1, 1, 0), (3, 7, 1), (65, 97, 0), (1030, 517, 3)):
        full = rng.randn(rows, width + shift).astype(dtype)
        tokens = tokens_of(rng, count, rows)
        a = D.Array.from_numpy(full)
        a = a[:, shift:] if shift else a
        check_rows(D.op.embedding(a, D.Array.from_numpy(tokens), 1.25).numpy(), full[:, shift:], tokens, 1.25)


def check_gradient(got, dy, tokens, rows, scale):
    dtype = dy.dtype.type
    want, size, n = np.zeros((rows, dy.shape[1]), np.longdouble), np.zeros((rows, dy.shape[1]), np.longdouble), np.zeros(rows)
    for i, t in enumerate(tokens):
        if 0 <= t < rows:
            want[t] += dy[i].astype(np.longdouble)
            size[t] += np.abs(dy[i].astype(np.longdouble))
            n[t] += 1
    assert (np.abs(got - want * scale) <= (n[:, None] + 1) * U[dtype] * size * abs(scale)).all()
    assert (got[n == 0] == 0).all()


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_gradient(gpu, D, rng, width, dtype):
    for count, rows, shift in ((1, 1, 0), (3, 7, 1), (63, 3, 0), (64, 1, 0), (65, 97, 0), (1030, 517, 3), (700, 2, 0)):
        full = rng.randn(count, width + shift).astype(dtype)
        tokens = tokens_of(rng, count, rows)
        a = D.Array.from_numpy(full)
        a = a[:, shift:] if shift else a
        got = D.op.embedding_backward(a, D.Array.from_numpy(tokens), rows, -0.75)
        assert got.shape == (rows, width)
        check_gradient(got.numpy(), full[:, shift:], tokens, rows, -0.75)


@pytest.mark.parametrize("count,rows", [(16384, 40000), (16385, 40000), (40000, 300), (70001, 65537), (20000, 1), (9000, 70000)])
def test_many_tokens(gpu, D, rng, count, rows):
    dy, tokens = rng.randn(count, 12).astype(np.float32), tokens_of(rng, count, rows)
    check_gradient(D.op.embedding_backward(D.Array.from_numpy(dy), D.Array.from_numpy(tokens), rows).numpy(), dy, tokens, rows, 1.0)


def test_one_token_throughout(gpu, D, rng):
    dy = rng.randn(5000, 70).astype(np.float32)
    for token in (0, 3, 9):
        tokens = np.full(5000, token, np.int32)
        check_gradient(D.op.embedding_backward(D.Array.from_numpy(dy), D.Array.from_numpy(tokens), 10).numpy(), dy, tokens, 10, 1.0)
    got = D.op.embedding_backward(D.Array.from_numpy(dy), D.Array.from_numpy(np.full(5000, -1, np.int32)), 10)
    assert (got.numpy() == 0).all()


def test_rows_of_padding_may_hold_anything(gpu, D, rng):
    dy, tokens = rng.randn(300, 33).astype(np.float32), tokens_of(rng, 300, 20)
    outside = (tokens < 0) | (tokens >= 20)
    dy[outside] = np.nan
    check_gradient(D.op.embedding_backward(D.Array.from_numpy(dy), D.Array.from_numpy(tokens), 20).numpy(), np.where(outside[:, None], 0, dy).astype(np.float32), tokens, 20, 1.0)


def test_shapes_destinations_and_order(gpu, D, rng):
    op = D.op
    table, tokens = rng.randn(50, 24).astype(np.float32), tokens_of(rng, 60, 50).reshape(4, 15)
    y = D.Array.empty((4, 15, 24))
    assert op.embedding(D.Array.from_numpy(table), D.Array.from_numpy(tokens), 2.0, out=y) is y
    check_rows(y.numpy().reshape(60, 24), table, tokens.reshape(-1), 2.0)
    # a lazily built table, and transposed views of both operands
    lazy = op.embedding(D.Array.from_numpy(table) * 3.0, D.Array.from_numpy(tokens))
    check_rows(lazy.numpy().reshape(60, 24), table * np.float32(3), tokens.reshape(-1), 1.0)
    turned = op.embedding(D.Array.from_numpy(np.ascontiguousarray(table.T)).T, D.Array.from_numpy(np.ascontiguousarray(tokens.T)).T)
    assert np.array_equal(turned.numpy().reshape(60, 24), op.embedding(D.Array.from_numpy(table), D.Array.from_numpy(tokens)).numpy().reshape(60, 24))
    # (an array made from a number has one axis; one value of an array has none)
    seven = D.Array.from_numpy(np.array([7], np.int32))
    for one, shape in ((op.embedding(D.Array.from_numpy(table), seven), (1, 24)), (op.embedding(D.Array.from_numpy(table), seven[0]), (24,))):
        assert one.shape == shape and np.array_equal(one.numpy().reshape(24), table[7])
    # the same bits every time, whatever lay in the destination
    dy = D.Array.from_numpy(rng.randn(4, 15, 24).astype(np.float32))
    out = D.Array.from_numpy(np.full((50, 24), np.nan, np.float32))
    first = op.embedding_backward(dy, D.Array.from_numpy(tokens), 50, out=out).numpy()
    assert np.array_equal(first, op.embedding_backward(dy, D.Array.from_numpy(tokens), 50).numpy())
    check_gradient(first, dy.numpy().reshape(60, 24), tokens.reshape(-1), 50, 1.0)


def test_no_tokens(gpu, D):
    got = D.op.embedding_backward(D.Array.empty((0, 8)), D.Array.empty((0,), D.DTYPE_INT32), 5)
    assert got.shape == (5, 8) and (got.numpy() == 0).all()


@pytest.mark.parametrize("count", [2000, 20000])
def test_recorded_and_replayed(gpu, D, rng, count):
    op = D.op
    table, tokens = D.Array.from_numpy(rng.randn(500, 40).astype(np.float32)), D.Array.from_numpy(tokens_of(rng, count, 500))
    dy, y, dtable = D.Array.from_numpy(rng.randn(count, 40).astype(np.float32)), D.Array.empty((count, 40)), D.Array.empty((500, 40))
    rec = D.Recording()
    with rec:
        op.embedding(table, tokens, 0.5, out=y)
        op.embedding_backward(dy, tokens, 500, 0.5, out=dtable)
    rec.make_graph()
    for _ in range(3):
        other = tokens_of(rng, count, 500)
        tokens.assign(D.Array.from_numpy(other))
        dy.assign(dy * -0.5)
        y.assign(y * 0.0), dtable.assign(dtable * 0.0)
        op.embedding_backward(dy * 1.0, D.Array.from_numpy(other[::-1].copy()), 500).numpy()  # the program's own work in between
        rec.replay()
        check_rows(y.numpy(), table.numpy(), other, 0.5)
        check_gradient(dtable.numpy(), dy.numpy(), other, 500, 0.5)

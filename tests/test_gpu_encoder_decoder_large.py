"""The operators of an encoder-decoder model on arrays whose bytes pass 2^32: what lies at their ends among zeros, whose results are known."""
import numpy as np
import pytest

from test_gpu_language_large import with_last_rows

pytestmark = pytest.mark.gpu


def end(a, rows):
    return a[a.shape[0] - rows:].ascontiguousarray().numpy()


def test_embedding(gpu, D, rng):
    A, op, width, rows = D.Array.from_numpy, D.op, 512, 2200000
    last = rng.randn(5, width).astype(np.float32)
    table = with_last_rows(D, rows, last)
    tokens = np.array([rows - 1, 0, rows - 5, -1, rows, rows - 2], np.int32)
    y = op.embedding(table, A(tokens), 2.0).numpy()
    assert np.array_equal(y, np.stack([2 * last[4], 0 * last[0], 2 * last[0], 0 * last[0], 0 * last[0], 2 * last[3]]))
    dy = rng.randn(6, width).astype(np.float32)
    dtable = op.embedding_backward(A(dy), A(tokens), rows, 2.0, out=table)
    assert np.array_equal(end(dtable, 6), np.stack([0 * dy[0], 2 * dy[2], 0 * dy[0], 0 * dy[0], 2 * dy[5], 2 * dy[0]]))
    del table, dtable
    # rows of dy, and positions, past 2^32 bytes
    many = np.full(rows, 3, np.int32)
    many[:-5] = -1
    got = op.embedding_backward(with_last_rows(D, rows, last), A(many), 7).numpy()
    assert np.abs(got[3] - last.astype(np.float64).sum(0)).max() <= 5 * 2.0 ** -24 * np.abs(last).sum(0).max() and not np.delete(got, 3, 0).any()


@pytest.mark.parametrize("queries,width", [(1, 64), (40, 64), (1, 128), (40, 128)])
def test_cross_attention(gpu, D, rng, queries, width):
    """All states but the last are zeros: scores 0 and values 0. With the last one's score s: y = e^s / (n - 1 + e^s) v, lse = ln(n - 1 + e^s)."""
    A, op, n = D.Array.from_numpy, D.op, 1100000000 // width
    k_last, v_last = rng.randn(1, width).astype(np.float32), rng.randn(1, width).astype(np.float32)
    q = rng.randn(1, queries, 1, width).astype(np.float32)
    q *= (18 / (q[0, :, 0] @ k_last[0]))[None, :, None, None]
    k, v = (with_last_rows(D, n, a).reshape(1, n, 1, width) for a in (k_last, v_last))
    y, lse = op.cross_attention(A(q), k, v, None, 1.0)
    s = q[0, :, 0].astype(np.float64) @ k_last[0].astype(np.float64)
    total = n - 1 + np.exp(s)
    p = np.exp(s) / total
    # (a score is off by (width + 4) u of its magnitudes, a weight by that; n equal weights of 1 or less are summed in runs of at most 32 n / 32 terms over thousands of lanes and
    # parts: by at most 2^-24 of the sum so far for every one of the slabs that a lane walks, fewer than 2^15, which is 2^-9 at worst)
    size = (np.abs(q[0, :, 0]) @ np.abs(k_last[0])) * (width + 4) * 2.0 ** -23
    assert (np.abs(lse.numpy()[0, :, 0] - np.log(total)) <= size + 2.0 ** -9).all()
    assert (np.abs(y.numpy()[0, :, 0] - p[:, None] * v_last) <= (2 * size + 2.0 ** -8)[:, None] * np.abs(v_last)).all()
    dy = rng.randn(*q.shape).astype(np.float32)
    dq, dk, dv = op.cross_attention_backward(A(dy), A(q), k, v, y, lse, None, 1.0)
    g, level, yy = dy[0, :, 0].astype(np.float64), lse.numpy()[0, :, 0].astype(np.float64), y.numpy()[0, :, 0].astype(np.float64)
    weight = np.exp(s - level)
    ds = weight * (g @ v_last[0] - (g * yy).sum(1))
    off = (2 * size + (width + 40) * 2.0 ** -22 * (1 + np.abs(level)))[:, None]
    magnitude = weight * (np.abs(g) @ np.abs(v_last[0]) + np.abs(g * yy).sum(1))
    assert (np.abs(dv.reshape(n, width)[n - 1].ascontiguousarray().numpy() - weight @ g) <= (off * weight[:, None] * np.abs(g)).sum(0)).all()
    assert (np.abs(dk.reshape(n, width)[n - 1].ascontiguousarray().numpy() - ds @ q[0, :, 0]) <= (off * magnitude[:, None] * np.abs(q[0, :, 0])).sum(0)).all()
    assert (np.abs(dq.numpy()[0, :, 0] - ds[:, None] * k_last) <= off * magnitude[:, None] * np.abs(k_last)).all()  # (the other states are zeros)


@pytest.mark.parametrize("rows", [3, 512])
def test_projected_cross_entropy(gpu, D, rng, rows):
    """A table of 2.2 million words as the projection, zeros but for the last: logits 0, and l for the last one."""
    A, op, inputs, vocab = D.Array.from_numpy, D.op, 500, 2200000
    last = rng.randn(1, inputs).astype(np.float32)
    x = rng.randn(rows, inputs).astype(np.float32)
    x *= (16 / (x @ last[0]))[:, None]
    table = with_last_rows(D, vocab, last)
    targets = np.full(rows, vocab - 1, np.int32)
    targets[0] = 7
    losses, lse = op.projected_cross_entropy(A(x), table.T, A(targets))
    l = x.astype(np.float64) @ last[0].astype(np.float64)
    want = np.log(vocab - 1 + np.exp(l))
    # (weights of 1 are summed exactly in segments, and the segments' sums in turn: fewer than 2^15 of them to a lane)
    size = (np.abs(x) @ np.abs(last[0])) * (inputs + 4) * 2.0 ** -23 + 2.0 ** -9
    assert (np.abs(lse.numpy() - want) <= size).all()
    assert (np.abs(losses.numpy() - (want - np.where(targets == 7, 0, l))) <= 2 * size).all()
    d = np.ones(rows, np.float32)
    dx, dw, _ = op.projected_cross_entropy_backward(A(d), A(x), table.T, A(targets), lse)
    g = np.exp(l - lse.numpy()) - (targets == vocab - 1)
    bound = 4 * size + 2.0 ** -18
    assert (np.abs(dx.numpy() - g[:, None] * last) <= bound[:, None] * np.abs(last)).all()
    assert (np.abs(dw.T[vocab - 1].ascontiguousarray().numpy() - g @ x) <= bound @ np.abs(x)).all()
    # row 0's target, and the weight that every word has
    small = np.exp(-lse.numpy().astype(np.float64))
    assert (np.abs(dw.T[7].ascontiguousarray().numpy() - (small @ x - x[0])) <= bound @ np.abs(x)).all()

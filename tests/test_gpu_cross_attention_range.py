"""Attention to an encoder's states: gradients that are cut into parts, values that bf16 pieces do not hold, two recordings in turn. Bounds as in test_gpu_cross_attention.py."""
import numpy as np
import pytest

from test_gpu_cross_attention import check_backward, check_forward, make

pytestmark = pytest.mark.gpu

# few tiles and many slabs of 32: the gradients' sums are formed in parts
PARTS = [(1, 700, 600, 2, 1, 64), (1, 300, 700, 4, 1, 128), (2, 600, 530, 1, 1, 200), (1, 1100, 90, 2, 2, 32), (2, 20, 1500, 2, 2, 256), (3, 513, 1025, 5, 1, 24)]


@pytest.mark.parametrize("size", PARTS, ids=str)
@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_parts(gpu, D, rng, size, dtype):
    q, k, v, counts = make(rng, dtype, *size)
    dy = rng.randn(*q.shape).astype(dtype)
    scale = 1 / np.sqrt(size[5])
    check_forward(D, q, k, v, counts, scale)
    first = [g.numpy() for g in check_backward(D, dy, q, k, v, counts, scale)]
    again = [g.numpy() for g in check_backward(D, dy, q, k, v, counts, scale)]
    assert all(np.array_equal(a, b) for a, b in zip(first, again))


def test_parts_of_a_padded_batch(gpu, D, rng):
    """Sequences without states, with one, and with all of them, in one call that is cut into parts."""
    for width in (64, 128, 256):
        q, k, v, counts = make(rng, np.float32, 4, 300, 650, 2, 1, width, [0, 1, 650, 33])
        check_backward(D, rng.randn(*q.shape).astype(np.float32), q, k, v, counts, 0.1)


@pytest.mark.parametrize("width", [20, 64, 100, 128, 200, 256])
@pytest.mark.parametrize("queries,keys", [(40, 70), (150, 200)])
def test_values_that_pieces_do_not_hold(gpu, D, rng, queries, keys, width):
    """Powers of two near the end of the type's range on one operand and their inverses on another: the results are the ordinary ones, times such a power. (A bound is a multiple of the
    magnitudes, so it moves with them; nothing is below the smallest normal number, 2^-126: the smallest factor is 2^-113 and what it multiplies, gradients of scores and weights, is
    compared where it is at least 2^-13 of its bound's size.)"""
    up, down = np.float32(2.0 ** 113), np.float32(2.0 ** -113)
    q, k, v, counts = make(rng, np.float32, 2, queries, keys, 2, 1, width, [keys, keys // 2])
    scale = 1 / np.sqrt(width)
    dy = rng.randn(*q.shape).astype(np.float32)
    check_forward(D, q, k, v * up, counts, scale)
    check_forward(D, q * up, k * down, v, counts, scale)
    check_forward(D, q * down, k * up, v, counts, scale)
    # one state of many: its tile alone is taken again
    some = v.copy()
    some[0, 3] *= up
    check_forward(D, q, k, some, counts, scale)
    A, op = D.Array.from_numpy, D.op
    y, lse = op.cross_attention(A(q), A(k), A(v), A(counts), scale)
    plain = [g.numpy() for g in op.cross_attention_backward(A(dy), A(q), A(k), A(v), y, lse, A(counts), scale)]
    check_backward(D, dy, q, k, v, counts, scale)
    for factors in ((up, 1, 1), (1, up, down), (1, down, up)):  # of dy, of q, of k
        yb, lb = op.cross_attention(A(q * factors[1]), A(k * factors[2]), A(v), A(counts), scale)
        got = op.cross_attention_backward(A(dy * factors[0]), A(q * factors[1]), A(k * factors[2]), A(v), yb, lb, A(counts), scale)
        for g, p, factor in zip(got, plain, (factors[0] * factors[2], factors[0] * factors[1], factors[0])):
            off = np.abs(g.numpy().astype(np.float64) / np.float64(factor) - p)
            # (both are off by rounding alone: weights by 2 (width + 4) u of scores of order |q| |k| scale < 10 and sums of `keys` or `rows` terms)
            assert off.max() <= 64 * (width + keys + 2 * queries) * 2.0 ** -24 * np.abs(p).max()


def test_infinite_values_stay_with_their_rows(gpu, D, rng):
    """A score of -inf has no weight; an infinite value is met by every row that gives its state weight, in its own column alone."""
    A, op = D.Array.from_numpy, D.op
    for width in (64, 128):
        q, k, v, counts = make(rng, np.float32, 2, 50, 90, 2, 2, width, [90, 60])
        v[0, 5, 1, 7] = np.inf
        y, lse = (a.numpy() for a in op.cross_attention(A(q), A(k), A(v), A(counts), 0.1))
        assert np.isfinite(lse).all() and (y[0, :, 1, 7] == np.inf).all()
        y[0, :, 1, 7] = 0
        assert np.isfinite(y).all()
        v[0, 5, 1, 7] = 0
        k[1, 10, 0, 3], q[1, :, 0, 3] = -np.inf, 1.0
        y, lse = (a.numpy() for a in op.cross_attention(A(q), A(k), A(v), A(counts), 0.1))
        assert np.isfinite(lse).all() and np.isfinite(y).all()
        finite = np.delete(k, 10, 1)
        check = op.cross_attention(A(q[1:]), A(finite[1:]), A(np.delete(v, 10, 1)[1:]), A(np.array([59], np.int32)), 0.1)
        assert np.abs(check[0].numpy()[0, :, 0] - y[1, :, 0]).max() < 1e-4


def test_two_recordings_in_turn(gpu, D, rng):
    """Single positions, whose parts meet by a counter, and gradients in parts: each recording has its own workspace."""
    A, op = D.Array.from_numpy, D.op
    held = []
    for size in ((2, 1, 2100, 4, 1, 64), (1, 400, 700, 2, 1, 128)):
        q, k, v, counts = make(rng, np.float32, *size)
        dy = rng.randn(*q.shape).astype(np.float32)
        ins = [A(a) for a in (dy, q, k, v, counts)]
        outs = [D.Array.empty(s) for s in (q.shape, q.shape[:3], q.shape, k.shape, k.shape)]
        rec = D.Recording()
        with rec:
            op.cross_attention(ins[1], ins[2], ins[3], ins[4], 0.1, out=outs[:2])
            op.cross_attention_backward(ins[0], ins[1], ins[2], ins[3], outs[0], outs[1], ins[4], 0.1, out=outs[2:])
        rec.make_graph()
        held.append((ins, outs, rec, (dy, q, k, v, counts)))
    for turn in range(3):
        for ins, outs, rec, data in held:
            ins[1].assign(ins[1] * -0.9)
            for o in outs:
                o.assign(o * 0.0)
        for ins, outs, rec, data in held:
            rec.replay()
            op.cross_attention(ins[1] * 2.0, ins[2], ins[3], ins[4])[0].numpy()  # the program's own work in between
        for ins, outs, rec, (dy, _, k, v, counts) in held:
            q = ins[1].numpy()
            check_forward(D, q, k, v, counts, 0.1, outs[:2])
            check_backward(D, dy, q, k, v, counts, 0.1, outs[2:])

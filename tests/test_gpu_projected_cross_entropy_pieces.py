"""Cross entropy of a projection whose logits are formed in several pieces of the vocabulary and blocks of rows. Bounds as in test_gpu_projected_cross_entropy.py.

A call goes by images (test_gpu_projected_cross_entropy_images.py) in fp32 from 512 rows and 256 tiles of 128 x 128 on, else by pieces of at most 128 MiB of logits for blocks of at
most 16384 rows; with one piece and up to 1024 rows a row's segments are joined by the launch that forms them, else by another. The sizes below keep to the latter."""
import numpy as np
import pytest

from test_gpu_projected_cross_entropy import case, check_forward, check_gradients

pytestmark = pytest.mark.gpu

F, G = np.float32, np.float64
# a second launch joins; two blocks; two pieces; both. With bias and rows of w, or without bias and columns
CASES = [(F, 1100, 24, 90, True, False), (F, 1100, 24, 90, False, True), (F, 2050, 5, 1030, True, True), (F, 16500, 7, 90, True, False), (F, 16500, 7, 90, False, True),
         (F, 400, 12, 90001, True, False), (F, 400, 12, 90001, False, True), (G, 1100, 24, 130, True, False), (G, 1100, 5, 16001, True, False), (G, 16500, 6, 130, True, False),
         (G, 16500, 3, 1100, False, True)]


@pytest.mark.parametrize("dtype,rows,inputs,vocab,biased,by_columns", CASES)
def test_both_directions(gpu, D, rng, dtype, rows, inputs, vocab, biased, by_columns):
    A, op = D.Array.from_numpy, D.op
    x, w, bias, targets = case(rng, dtype, rows, inputs, vocab)
    b, wa = A(bias) if biased else None, A(np.ascontiguousarray(w.T)).T if by_columns else A(w)
    bias = bias if biased else None
    losses, lse = op.projected_cross_entropy(A(x), wa, A(targets), b)
    check_forward(x, w, bias, targets, losses.numpy(), lse.numpy())
    d = rng.randn(rows).astype(dtype)
    got = op.projected_cross_entropy_backward(A(d), A(x), wa, A(targets), lse, b)
    check_gradients(d, x, w, bias, targets, lse.numpy(), got)
    there = (targets >= 0) & (targets < vocab)
    assert (got[0].numpy()[~there] == 0).all()


def test_recorded_and_replayed(gpu, D, rng):
    A, op = D.Array.from_numpy, D.op
    rows, inputs, vocab = 400, 3, 90001
    x, w, bias, targets = case(rng, F, rows, inputs, vocab)
    d = rng.randn(rows).astype(F)
    xa, wa, ba, ta, da = A(x), A(w), A(bias), A(targets), A(d)
    outs = [D.Array.empty(s) for s in ((rows,), (rows,), x.shape, w.shape, bias.shape)]
    rec = D.Recording()
    with rec:
        op.projected_cross_entropy(xa, wa, ta, ba, out=outs[:2])
        op.projected_cross_entropy_backward(da, xa, wa, ta, outs[1], ba, out=outs[2:])
    rec.make_graph()
    for _ in range(3):
        xa.assign(xa * -0.8)
        for o in outs:
            o.assign(o * 0.0)
        op.projected_cross_entropy(xa * 2.0, wa, ta)[0].numpy()  # the program's own work in between
        rec.replay()
        check_forward(xa.numpy(), w, bias, targets, outs[0].numpy(), outs[1].numpy())
        check_gradients(d, xa.numpy(), w, bias, targets, outs[1].numpy(), outs[2:])


def test_a_masked_piece(gpu, D, rng):
    """A piece of the vocabulary that the bias takes out whole, with targets in the other."""
    A, op = D.Array.from_numpy, D.op
    rows, inputs, vocab = 1100, 6, 16001
    for dtype, n in ((G, 1100), (F, 400)):
        vocab = 16001 if dtype == G else 90001
        x, w, bias, targets = case(rng, dtype, n, inputs, vocab, outside=False)
        d = rng.randn(n).astype(dtype)
        for out in (slice(0, 85000 if dtype == F else 15000), slice(14000 if dtype == G else 80000, None)):
            b = bias.copy()
            b[out] = -np.inf
            kept = np.flatnonzero(np.isfinite(b))
            t = rng.choice(kept, n).astype(np.int32)
            named = np.searchsorted(kept, t).astype(np.int32)
            losses, lse = op.projected_cross_entropy(A(x), A(w), A(t), A(b))
            check_forward(x, w[:, kept], b[kept], named, losses.numpy(), lse.numpy())
            dx, dw, dbias = op.projected_cross_entropy_backward(A(d), A(x), A(w), A(t), lse, A(b))
            check_gradients(d, x, w[:, kept], b[kept], named, lse.numpy(), (dx, None, None))
            assert (dw.numpy()[:, out] == 0).all() and (dbias.numpy()[out] == 0).all()

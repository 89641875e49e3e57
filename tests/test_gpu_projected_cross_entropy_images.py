"""Cross entropy of a projection where rows and vocabulary are many: fp32 values cut into pieces beforehand, the softmax at the ends of the products. Against the formulas in 64 bits."""
import numpy as np
import pytest

from test_gpu_projected_cross_entropy import case, check_forward, check_gradients, gradients

pytestmark = pytest.mark.gpu

# (from 512 rows and 256 tiles of 128 x 128 on)
SIZES = [(512, 16, 8192), (513, 17, 8193), (511, 20, 8300), (640, 33, 6600), (2049, 1, 2050), (600, 130, 7001), (4200, 15, 1000)]


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("biased", [True, False])
def test_both_directions(gpu, D, rng, size, biased):
    A, op = D.Array.from_numpy, D.op
    x, w, bias, targets = case(rng, np.float32, *size)
    b = A(bias) if biased else None
    losses, lse = op.projected_cross_entropy(A(x), A(w), A(targets), b)
    check_forward(x, w, bias if biased else None, targets, losses.numpy(), lse.numpy())
    d = rng.randn(size[0]).astype(np.float32)
    got = op.projected_cross_entropy_backward(A(d), A(x), A(w), A(targets), lse, b)
    check_gradients(d, x, w, bias if biased else None, targets, lse.numpy(), got)
    there = (targets >= 0) & (targets < size[2])
    assert (got[0].numpy()[~there] == 0).all()


def test_several_pieces_and_blocks(gpu, D, rng):
    """More rows than a block has, and more columns than the image of a block's gradient of logits."""
    A, op = D.Array.from_numpy, D.op
    x, w, bias, targets = case(rng, np.float32, 16500, 18, 5300)
    losses, lse = op.projected_cross_entropy(A(x), A(w), A(targets), A(bias))
    check_forward(x, w, bias, targets, losses.numpy(), lse.numpy())
    d = (rng.rand(16500) + 0.5).astype(np.float32)
    got = op.projected_cross_entropy_backward(A(d), A(x), A(w), A(targets), lse, A(bias))
    check_gradients(d, x, w, bias, targets, lse.numpy(), got)


def test_views_and_destinations(gpu, D, rng):
    A, op = D.Array.from_numpy, D.op
    size = (520, 37, 7003)
    x, w, bias, targets = case(rng, np.float32, *size)
    d = rng.randn(size[0]).astype(np.float32)
    table, wider = A(np.ascontiguousarray(w.T)), A(np.concatenate([w, w], 1))
    for xa, wa in ((A(x), table.T), (A(x), wider[:, :size[2]]), (A(np.concatenate([x, x], 1))[:, size[1]:], A(w))):
        losses, lse = op.projected_cross_entropy(xa, wa, A(targets), A(bias))
        check_forward(x, w, bias, targets, losses.numpy(), lse.numpy())
        got = op.projected_cross_entropy_backward(A(d), xa, wa, A(targets), lse, A(bias))
        check_gradients(d, x, w, bias, targets, lse.numpy(), got)
    dtable = A(np.full((size[2], size[1]), np.nan, np.float32))
    outs = (A(np.full(x.shape, np.nan, np.float32)), dtable.T, A(np.full(size[2], np.nan, np.float32)))
    got = op.projected_cross_entropy_backward(A(d), A(x), A(w), A(targets), lse, A(bias), out=outs)
    check_gradients(d, x, w, bias, targets, lse.numpy(), got)
    got = op.projected_cross_entropy_backward(A(d), A(x), table.T, A(targets), lse, A(bias), out=(None, A(np.full(w.shape, np.nan, np.float32)), None))
    check_gradients(d, x, w, bias, targets, lse.numpy(), got)


def test_rows_without_a_target_may_hold_anything(gpu, D, rng):
    A, op = D.Array.from_numpy, D.op
    x, w, bias, targets = case(rng, np.float32, 530, 40, 7000, outside=False)
    out = [1, 40, 500, 529]
    targets[out] = [-1, 7000, -5, 2 ** 31 - 1]
    keep = (targets >= 0) & (targets < 7000)
    d = rng.randn(530).astype(np.float32)
    for bad in (np.nan, np.inf, np.float32(3.4e38)):
        dirty, dd = x.copy(), d.copy()
        dirty[out], dd[out] = bad, bad
        losses, lse = op.projected_cross_entropy(A(dirty), A(w), A(targets), A(bias))
        assert (losses.numpy()[~keep] == 0).all()
        check_forward(x[keep], w, bias, targets[keep], losses.numpy()[keep], lse.numpy()[keep])
        got = op.projected_cross_entropy_backward(A(dd), A(dirty), A(w), A(targets), lse, A(bias))
        check_gradients(d, x, w, bias, targets, np.where(keep, lse.numpy(), 0), got)
        assert (got[0].numpy()[~keep] == 0).all()


def test_a_masked_vocabulary(gpu, D, rng):
    A, op = D.Array.from_numpy, D.op
    x, w, bias, targets = case(rng, np.float32, 512, 24, 8200, outside=False)
    d = rng.randn(512).astype(np.float32)
    out = rng.rand(8200) < 0.5
    out[:2048] = True
    targets[:] = rng.choice(np.flatnonzero(~out), 512)
    named = np.searchsorted(np.flatnonzero(~out), targets).astype(np.int32)
    for mask in (-np.inf, np.finfo(np.float32).min):
        bias[out] = mask
        losses, lse = op.projected_cross_entropy(A(x), A(w), A(targets), A(bias))
        check_forward(x, w[:, ~out], bias[~out], named, losses.numpy(), lse.numpy())
        dx, dw, dbias = op.projected_cross_entropy_backward(A(d), A(x), A(w), A(targets), lse, A(bias))
        assert (dw.numpy()[:, out] == 0).all() and (dbias.numpy()[out] == 0).all()
        check_gradients(d, x, w[:, ~out], bias[~out], named, lse.numpy(), (dx,))
    bias[:] = -np.inf
    losses, lse = op.projected_cross_entropy(A(x), A(w), A(targets), A(bias))
    assert (losses.numpy() == np.inf).all() and (lse.numpy() == -np.inf).all()
    for g in op.projected_cross_entropy_backward(A(d), A(x), A(w), A(targets), lse, A(bias)):
        assert (g.numpy() == 0).all()


def test_values_that_pieces_do_not_hold(gpu, D, rng):
    """Values at the end of the type's range, sums of them that pass it, infinities and NaN: what the fp32 products give."""
    A, op = D.Array.from_numpy, D.op
    x, w, bias, targets = case(rng, np.float32, 512, 24, 8200, outside=False)
    huge = x.copy()
    huge[7] = 0
    huge[7, 3] = np.finfo(np.float32).max  # (rounded to eight bits it would be infinite)
    small = w.copy()
    small[3] = rng.randn(8200) * 1e-38
    losses, lse = op.projected_cross_entropy(A(huge), A(small), A(targets), A(bias))
    check_forward(huge, small, bias, targets, losses.numpy(), lse.numpy())
    # a column of -inf on positive rows is as good as a mask
    x, masked = np.abs(x), w.copy()
    masked[:, 4000] = -np.inf
    targets[targets == 4000] = 4001
    losses, lse = op.projected_cross_entropy(A(x), A(masked), A(targets), A(bias))
    keep = np.arange(8200) != 4000
    check_forward(x, w[:, keep], bias[keep], (targets - (targets > 4000)).astype(np.int32), losses.numpy(), lse.numpy())
    # a row of NaN is alone
    x[2] = np.nan
    losses, lse = op.projected_cross_entropy(A(x), A(w), A(targets), A(bias))
    rest = np.arange(512) != 2
    assert np.isnan(losses.numpy()[2]) and np.isnan(lse.numpy()[2])
    check_forward(x[rest], w, bias, targets[rest], losses.numpy()[rest], lse.numpy()[rest])
    d = rng.randn(512).astype(np.float32)
    dx = op.projected_cross_entropy_backward(A(d), A(x), A(w), A(targets), lse, A(bias))[0].numpy()
    assert np.isnan(dx[2]).all() and np.isfinite(dx[rest]).all()


def test_small_gradients_keep_their_digits(gpu, D, rng):
    """Weights of e^-75 to e^-90 and gradients of losses of 1e-2, in columns that no row names. The exponential gives 0 below the smallest normal number, 2^-126 (e^-87.3), which a
    row's gradient of a logit may be off by, times d; and d p is rounded to a multiple of 2^-149."""
    A, op = D.Array.from_numpy, D.op
    x, w, bias, targets = case(rng, np.float32, 512, 24, 8200, outside=False)
    targets %= 4000
    bias[4000:] -= 75.0
    losses, lse = op.projected_cross_entropy(A(x), A(w), A(targets), A(bias))
    check_forward(x, w, bias, targets, losses.numpy(), lse.numpy())
    d = np.full(512, 1e-2, np.float32)
    got = op.projected_cross_entropy_backward(A(d), A(x), A(w), A(targets), lse, A(bias))
    off = 1e-2 * 2.0 ** -126 + 2.0 ** -150
    for g, (want, bound), more in zip(got, gradients(d, x, w, bias, targets, lse.numpy()), (off * np.abs(w).sum(1), off * np.abs(x).sum(0)[:, None], off * 512)):
        assert (np.abs(g.numpy() - want) <= bound + more).all()


def test_recorded_and_replayed(gpu, D, rng):
    """Two recordings, each with its own workspace, replayed in turn."""
    A, op = D.Array.from_numpy, D.op
    x, w, bias, targets = case(rng, np.float32, 530, 40, 7000)
    d = rng.randn(530).astype(np.float32)
    wa, ba, ta, da = A(w), A(bias), A(targets), A(d)
    held = []
    for factor in (1.0, -0.7):
        xa = A((x * factor).astype(np.float32))
        outs = [D.Array.empty(s) for s in ((530,), (530,), x.shape, w.shape, bias.shape)]
        rec = D.Recording()
        with rec:
            op.projected_cross_entropy(xa, wa, ta, ba, out=outs[:2])
            op.projected_cross_entropy_backward(da, xa, wa, ta, outs[1], ba, out=outs[2:])
        rec.make_graph()
        held.append((xa, outs, rec))
    for _ in range(3):
        for xa, outs, rec in held:
            xa.assign(xa * -0.8)
            for o in outs:
                o.assign(o * 0.0)
        for xa, outs, rec in held:
            rec.replay()
            op.projected_cross_entropy(xa * 2.0, wa, ta)[0].numpy()  # the program's own work in between
        for xa, outs, rec in held:
            check_forward(xa.numpy(), w, bias, targets, outs[0].numpy(), outs[1].numpy())
            check_gradients(d, xa.numpy(), w, bias, targets, outs[1].numpy(), outs[2:])


def test_the_same_bits_twice(gpu, D, rng):
    A, op = D.Array.from_numpy, D.op
    x, w, bias, targets = case(rng, np.float32, 700, 100, 7000)
    d = A(rng.randn(700).astype(np.float32))
    xa, wa, ba, ta = A(x), A(w), A(bias), A(targets)
    first = None
    for _ in range(3):
        losses, lse = op.projected_cross_entropy(xa, wa, ta, ba)
        got = [losses.numpy(), lse.numpy()] + [g.numpy() for g in op.projected_cross_entropy_backward(d, xa, wa, ta, lse, ba)]
        first = first or got
        assert all(np.array_equal(a, b) for a, b in zip(first, got))

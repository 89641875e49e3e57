"""Cross entropy of a projection with infinite operands: rows that their own infinities leave without weight, columns of w that are out. Bounds as in test_gpu_projected_cross_entropy.py."""
import numpy as np
import pytest

from test_gpu_projected_cross_entropy import case, check_forward, check_gradients, gradients

pytestmark = pytest.mark.gpu

# The last one goes by images, which fp64 never does
SIZES = [(6, 40, 300), (150, 96, 700), (530, 40, 7000)]
KINDS = [(s, t) for s in SIZES for t in (np.float32, np.float64) if s != SIZES[-1] or t == np.float32]


@pytest.mark.parametrize("size,dtype", KINDS, ids=str)
@pytest.mark.parametrize("by_columns", [False, True])
def test_rows_whose_infinities_leave_no_weight(gpu, D, rng, size, dtype, by_columns):
    """x holds -inf where w is positive: every logit of the row is -inf. It has no part in the gradients, as if it had no target."""
    A, op = D.Array.from_numpy, D.op
    x, w, bias, targets = case(rng, dtype, *size, outside=False)
    w[2] = np.abs(w[2]) + dtype(0.1)
    out = [0, size[0] - 2]
    dirty = x.copy()
    dirty[out, 2] = -np.inf
    wa = A(np.ascontiguousarray(w.T)).T if by_columns else A(w)
    losses, lse = op.projected_cross_entropy(A(dirty), wa, A(targets), A(bias))
    assert (losses.numpy()[out] == np.inf).all() and (lse.numpy()[out] == -np.inf).all()
    keep = np.ones(size[0], bool)
    keep[out] = False
    check_forward(x[keep], w, bias, targets[keep], losses.numpy()[keep], lse.numpy()[keep])
    d = rng.randn(size[0]).astype(dtype)
    got = op.projected_cross_entropy_backward(A(d), A(dirty), wa, A(targets), lse, A(bias))
    check_gradients(d, x, w, bias, np.where(keep, targets, -1), np.where(keep, lse.numpy(), 0), got)
    assert (got[0].numpy()[out] == 0).all()


@pytest.mark.parametrize("size,dtype", KINDS, ids=str)
def test_columns_of_infinities(gpu, D, rng, size, dtype):
    """A word whose column of w is -inf in one place is out where x is positive: lse, losses, dw and dbias are those without it. Its weight of 0 times -inf makes NaN of dx
    in that place of a row, there alone."""
    A, op = D.Array.from_numpy, D.op
    x, w, bias, targets = case(rng, dtype, *size)
    x[:, 1] = np.abs(x[:, 1]) + dtype(0.1)
    targets[targets == 5] = 4
    masked, keep = w.copy(), np.arange(size[2]) != 5
    masked[1, 5] = -np.inf
    losses, lse = op.projected_cross_entropy(A(x), A(masked), A(targets), A(bias))
    named = np.where(targets > 5, targets - 1, targets).astype(np.int32)
    check_forward(x, w[:, keep], bias[keep], named, losses.numpy(), lse.numpy())
    d = rng.randn(size[0]).astype(dtype)
    dx, dw, dbias = (g.numpy() for g in op.projected_cross_entropy_backward(A(d), A(x), A(masked), A(targets), lse, A(bias)))
    assert (dw[:, 5] == 0).all() and dbias[5] == 0
    assert np.isnan(dx[:, 1]).all()
    others = np.arange(size[1]) != 1
    want = [(w_[:, others] if i == 0 else w_) for i, w_ in enumerate((dx, dw[:, keep], dbias[keep]))]
    bounds = gradients(d, x, w[:, keep], bias[keep], named, lse.numpy())
    for i, (got, (exact, bound)) in enumerate(zip(want, bounds)):
        if i == 0:
            exact, bound = exact[:, others], bound[:, others]
        assert (np.abs(got - exact) <= bound).all()


@pytest.mark.parametrize("size,dtype", KINDS, ids=str)
def test_a_logit_of_plus_infinity_makes_its_row_nan(gpu, D, rng, size, dtype):
    A = D.Array.from_numpy
    x, w, bias, targets = case(rng, dtype, *size, outside=False)
    w[2] = np.abs(w[2]) + dtype(0.1)
    dirty = x.copy()
    dirty[3, 2] = np.inf
    losses, lse = (a.numpy() for a in D.op.projected_cross_entropy(A(dirty), A(w), A(targets), A(bias)))
    assert np.isnan(losses[3]) and np.isnan(lse[3])
    keep = np.arange(size[0]) != 3
    check_forward(x[keep], w, bias, targets[keep], losses[keep], lse[keep])

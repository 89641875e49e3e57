"""Cross entropy of a projection whose logits are not kept, and its gradients, against the formulas in 64 bits: sizes around every change of the kernels, padding, views.

u is half a unit in the last place of 1. A logit is a sum of `inputs` products, each off by at most 2 u of its size, and a bias: off by at most (inputs + 4) u of the sum A of the
magnitudes. A weight e^(l - m) is off by twice that, by the rounding of l - m and by 4 u for the exponential, relative; a sum of `vocab` of them by vocab u more at most.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = {np.float32: 2.0 ** -24, np.float64: 2.0 ** -53}
# rows, inputs, vocabulary
SIZES = [(1, 1, 1), (1, 3, 2), (3, 5, 7), (2, 16, 63), (7, 33, 1024), (8, 64, 1025), (1, 100, 5001), (33, 20, 511), (64, 65, 513), (65, 70, 2048), (70, 129, 2049),
         (130, 128, 1000), (200, 31, 97), (300, 256, 1111), (129, 515, 1537), (1000, 80, 128)]


def case(rng, dtype, rows, inputs, vocab, outside=True):
    x, w, bias = rng.randn(rows, inputs).astype(dtype), (rng.randn(inputs, vocab) * 1.5 / np.sqrt(inputs)).astype(dtype), (0.3 * rng.randn(vocab)).astype(dtype)
    targets = rng.randint(0, vocab, rows).astype(np.int32)
    if outside and rows > 4:
        targets[rng.randint(rows)], targets[rng.randint(rows)] = -1, vocab
    return x, w, bias, targets


def logits_of(x, w, bias):
    wide = np.longdouble if x.dtype == np.float64 else np.float64
    b = 0 if bias is None else bias.astype(wide)
    return x.astype(wide) @ w.astype(wide) + b, np.abs(x.astype(wide)) @ np.abs(w.astype(wide)) + np.abs(b)


def check_forward(x, w, bias, targets, losses, lse):
    u, (rows, inputs), vocab = U[x.dtype.type], x.shape, w.shape[1]
    l, size = logits_of(x, w, bias)
    top = l.max(1)
    total = np.exp(l - top[:, None]).sum(1)
    want_lse = top + np.log(total)
    there = (targets >= 0) & (targets < vocab)
    want = np.where(there, want_lse - l[np.arange(rows), np.where(there, targets, 0)], 0)
    error = 3 * (inputs + 4) * u * size.max(1) + u * (l.max(1) - l.min(1)) + (vocab + 16) * u
    assert (np.abs(lse - want_lse) <= error + u * np.abs(want_lse) + u * np.abs(top)).all()
    assert (np.abs(losses - want) <= error + 3 * u * np.abs(want)).all()
    assert (losses[~there] == 0).all()


def gradients(d, x, w, bias, targets, lse):
    u, (rows, inputs), vocab = U[x.dtype.type], x.shape, w.shape[1]
    l, size = logits_of(x, w, bias)
    there = (targets >= 0) & (targets < vocab)
    level = lse.astype(l.dtype)[:, None]
    p = np.exp(l - level)
    hot = np.zeros_like(l)
    hot[np.arange(rows)[there], targets[there]] = 1
    given = np.where(there, d, 0).astype(l.dtype)[:, None]
    g = given * (p - hot)
    g_bound = np.abs(given) * (p * ((inputs + 4) * u * size + 2 * u * np.abs(l - level) + 6 * u) + 2 * u * np.abs(p - hot))
    x, w = x.astype(l.dtype), w.astype(l.dtype)
    return ((g @ w.T, (g_bound + (vocab + 8) * u * np.abs(g)) @ np.abs(w).T), (x.T @ g, np.abs(x).T @ (g_bound + (rows + 8) * u * np.abs(g))),
            (g.sum(0), (g_bound + (rows + 8) * u * np.abs(g)).sum(0)))


def check_gradients(d, x, w, bias, targets, lse, got):
    for g, (want, bound) in zip(got, gradients(d, x, w, bias, targets, lse)):
        if g is not None:
            assert g.shape == want.shape
            assert (np.abs(g.numpy() - want) <= bound).all(), (np.abs(g.numpy() - want) / np.maximum(bound, 1e-300)).max()


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("biased", [True, False])
def test_both_directions(gpu, D, rng, size, dtype, biased):
    A, op = D.Array.from_numpy, D.op
    x, w, bias, targets = case(rng, dtype, *size)
    b = A(bias) if biased else None
    losses, lse = op.projected_cross_entropy(A(x), A(w), A(targets), b)
    assert losses.shape == lse.shape == (size[0],)
    check_forward(x, w, bias if biased else None, targets, losses.numpy(), lse.numpy())
    d = rng.randn(size[0]).astype(dtype)
    got = op.projected_cross_entropy_backward(A(d), A(x), A(w), A(targets), lse, b)
    assert (got[2] is None) == (not biased)
    check_gradients(d, x, w, bias if biased else None, targets, lse.numpy(), got)
    there = (targets >= 0) & (targets < size[2])
    assert (got[0].numpy()[~there] == 0).all()


@pytest.mark.parametrize("rows,inputs,vocab", [(513, 256, 6000), (2100, 192, 17000), (17000, 40, 2500), (300, 1024, 9001)])
def test_pieces_and_blocks(gpu, D, rng, rows, inputs, vocab):
    A, op = D.Array.from_numpy, D.op
    x, w, bias, targets = case(rng, np.float32, rows, inputs, vocab)
    losses, lse = op.projected_cross_entropy(A(x), A(w), A(targets), A(bias))
    check_forward(x, w, bias, targets, losses.numpy(), lse.numpy())
    d = (rng.rand(rows) + 0.5).astype(np.float32)
    got = op.projected_cross_entropy_backward(A(d), A(x), A(w), A(targets), lse, A(bias))
    check_gradients(d, x, w, bias, targets, lse.numpy(), got)


@pytest.mark.parametrize("size", [(5, 24, 300), (150, 136, 1300)])
@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_views_and_destinations(gpu, D, rng, size, dtype):
    A, op = D.Array.from_numpy, D.op
    x, w, bias, targets = case(rng, dtype, *size)
    d = rng.randn(size[0]).astype(dtype)
    table, wider = A(np.ascontiguousarray(w.T)), A(np.concatenate([w, w], 1))
    for xa, wa in ((A(x), table.T), (A(x), wider[:, :size[2]]), (A(np.concatenate([x, x], 1))[:, size[1]:], A(w)), (A(np.ascontiguousarray(x.T)).T, A(w)),
                   (A(x[::-1].copy())[::-1], A(w) * 1.0)):
        losses, lse = op.projected_cross_entropy(xa, wa, A(targets), A(bias))
        check_forward(x, w, bias, targets, losses.numpy(), lse.numpy())
        got = op.projected_cross_entropy_backward(A(d), xa, wa, A(targets), lse, A(bias))
        check_gradients(d, x, w, bias, targets, lse.numpy(), got)
    # a table's gradient where the table lies as [vocabulary, inputs]
    dtable = A(np.full((size[2], size[1]), np.nan, dtype))
    outs = (A(np.full(x.shape, np.nan, dtype)), dtable.T, A(np.full(size[2], np.nan, dtype)))
    got = op.projected_cross_entropy_backward(A(d), A(x), table.T, A(targets), lse, A(bias), out=outs)
    assert got[0] is outs[0] and got[1] is outs[1] and got[2] is outs[2]
    check_gradients(d, x, w, bias, targets, lse.numpy(), got)
    assert np.array_equal(dtable.numpy(), got[1].numpy().T)
    outs = tuple(A(np.full(size[0], np.nan, dtype)) for _ in range(2))
    op.projected_cross_entropy(A(x), A(w), A(targets), A(bias), out=outs)
    check_forward(x, w, bias, targets, outs[0].numpy(), outs[1].numpy())
    # rows of more than one axis
    if size[0] % 5 == 0:
        shaped = op.projected_cross_entropy(A(x.reshape(5, -1, size[1])), A(w), A(targets.reshape(5, -1)), A(bias))
        assert shaped[0].shape == (5, size[0] // 5) and np.array_equal(shaped[0].numpy().reshape(-1), outs[0].numpy())
        back = op.projected_cross_entropy_backward(A(d.reshape(5, -1)), A(x.reshape(5, -1, size[1])), A(w), A(targets.reshape(5, -1)), shaped[1], A(bias))
        assert back[0].shape == (5, size[0] // 5, size[1])
        check_gradients(d, x, w, bias, targets, outs[1].numpy(), (back[0].reshape(size[0], size[1]),) + tuple(back[1:]))


@pytest.mark.parametrize("rows", [6, 140])
@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_rows_without_a_target_may_hold_anything(gpu, D, rng, rows, dtype):
    A, op = D.Array.from_numpy, D.op
    x, w, bias, targets = case(rng, dtype, rows, 96, 700, outside=False)
    targets[[1, rows - 1]] = [-1, 700]
    d = rng.randn(rows).astype(dtype)
    for bad in (np.nan, np.inf):
        dirty, dd = x.copy(), d.copy()
        dirty[[1, rows - 1]] = bad
        dd[[1, rows - 1]] = bad
        losses, lse = op.projected_cross_entropy(A(dirty), A(w), A(targets), A(bias))
        keep = targets < 700
        keep &= targets >= 0
        assert (losses.numpy()[~keep] == 0).all()
        check_forward(x[keep], w, bias, targets[keep], losses.numpy()[keep], lse.numpy()[keep])
        got = op.projected_cross_entropy_backward(A(dd), A(dirty), A(w), A(targets), lse, A(bias))
        clean = np.where(keep, lse.numpy(), 0)
        check_gradients(d, x, w, bias, targets, clean, got)
        assert (got[0].numpy()[~keep] == 0).all()


@pytest.mark.parametrize("rows", [4, 100])
@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_a_masked_vocabulary(gpu, D, rng, rows, dtype):
    """-inf and the type's lowest value in the bias take words out; with all of them out nothing is left."""
    A, op = D.Array.from_numpy, D.op
    x, w, bias, targets = case(rng, dtype, rows, 72, 1500, outside=False)
    d = rng.randn(rows).astype(dtype)
    out = rng.rand(1500) < 0.5
    out[:1024] = True  # (a whole segment)
    out[1400] = False
    targets[:] = rng.choice(np.flatnonzero(~out), rows)
    some = op.projected_cross_entropy(A(x), A(w[:, ~out].copy()), A(np.searchsorted(np.flatnonzero(~out), targets).astype(np.int32)), A(bias[~out]))
    for mask in (-np.inf, np.finfo(dtype).min):
        bias[out] = mask
        losses, lse = op.projected_cross_entropy(A(x), A(w), A(targets), A(bias))
        check_forward(x, w[:, ~out], bias[~out], np.searchsorted(np.flatnonzero(~out), targets).astype(np.int32), losses.numpy(), lse.numpy())
        dx, dw, dbias = op.projected_cross_entropy_backward(A(d), A(x), A(w), A(targets), lse, A(bias))
        assert (dw.numpy()[:, out] == 0).all() and (dbias.numpy()[out] == 0).all()
        check_gradients(d, x, w[:, ~out], bias[~out], np.searchsorted(np.flatnonzero(~out), targets).astype(np.int32), lse.numpy(), (dx,))
    bias[:] = -np.inf
    losses, lse = op.projected_cross_entropy(A(x), A(w), A(targets), A(bias))
    assert (losses.numpy() == np.inf).all() and (lse.numpy() == -np.inf).all()
    for g in op.projected_cross_entropy_backward(A(d), A(x), A(w), A(targets), lse, A(bias)):
        assert (g.numpy() == 0).all()


def test_a_row_that_is_not_finite_is_alone(gpu, D, rng):
    A = D.Array.from_numpy
    for rows in (5, 200):
        x, w, bias, targets = case(rng, np.float32, rows, 96, 900, outside=False)
        x[2] = np.nan
        losses, lse = D.op.projected_cross_entropy(A(x), A(w), A(targets), A(bias))
        assert np.isnan(losses.numpy()[2]) and np.isnan(lse.numpy()[2])
        keep = np.arange(rows) != 2
        check_forward(x[keep], w, bias, targets[keep], losses.numpy()[keep], lse.numpy()[keep])


def test_no_rows(gpu, D, rng):
    A, op = D.Array.from_numpy, D.op
    w, bias = A(rng.randn(8, 30).astype(np.float32)), A(rng.randn(30).astype(np.float32))
    none, whole, per_row = D.Array.empty((0, 8)), D.Array.empty((0,), D.DTYPE_INT32), D.Array.empty((0,))
    losses, lse = op.projected_cross_entropy(none, w, whole, bias)
    assert losses.shape == lse.shape == (0,)
    dx, dw, dbias = op.projected_cross_entropy_backward(per_row, none, w, whole, lse, bias)
    assert dx.shape == (0, 8) and (dw.numpy() == 0).all() and (dbias.numpy() == 0).all()


def test_gradients_against_differences(gpu, D, rng):
    """By central differences in double: the error of a step h is h^2 / 6 of a third derivative of order 1 and u / h of rounding: below 1e-6 at h = 1e-4."""
    A, op = D.Array.from_numpy, D.op
    x, w, bias, targets = case(rng, np.float64, 6, 5, 40)
    d = rng.randn(6)
    _, lse = op.projected_cross_entropy(A(x), A(w), A(targets), A(bias))
    grads = op.projected_cross_entropy_backward(A(d), A(x), A(w), A(targets), lse, A(bias))
    for which, g in enumerate(grads):
        for _ in range(12):
            at = tuple(rng.randint(n) for n in (x, w, bias)[which].shape)
            value = []
            for h in (1e-4, -1e-4):
                m = [x.copy(), w.copy(), bias.copy()]
                m[which][at] += h
                value.append((op.projected_cross_entropy(A(m[0]), A(m[1]), A(targets), A(m[2]))[0].numpy() * d).sum())
            assert abs((value[0] - value[1]) / 2e-4 - g.numpy()[at]) < 1e-6


@pytest.mark.parametrize("rows,inputs,vocab", [(4, 64, 3000), (300, 256, 5000)])
def test_recorded_and_replayed(gpu, D, rng, rows, inputs, vocab):
    A, op = D.Array.from_numpy, D.op
    x, w, bias, targets = case(rng, np.float32, rows, inputs, vocab)
    d = rng.randn(rows).astype(np.float32)
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

"""Attention to an encoder's states where values are extreme: scores whose partial sums pass what bf16 pieces hold, infinities in the last state. Bounds as in test_gpu_cross_attention.py."""
import numpy as np
import pytest

from test_gpu_cross_attention import check_backward, check_forward, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("width", [64, 100, 128, 200, 256])
@pytest.mark.parametrize("queries,keys", [(70, 90), (150, 700)])
@pytest.mark.parametrize("sign", [-1, 1])
def test_scores_whose_partial_sums_are_large(gpu, D, rng, width, queries, keys, sign):
    """The products of one state are 1.25 * 2^91 over 30 values of the width and the opposite over the next 30: every sum of them is exact in fp32 (a multiple of 1.25 * 2^91 of at most six
    bits) and the score 0, but halfway it passes 2^96. So the results are those of a state of zeros. (The scale is ln 2, which times log2 e is 1: operands stay powers of two.)"""
    q, k, v, counts = make(rng, np.float32, 2, queries, keys, 2, 1, width, [keys, keys // 2])
    large = np.arange(width) % 16 != 15  # (fifteen of every sixteen values; the others are ordinary ones)
    large[64:] = False
    ordinary = ~large
    q[..., large], k[..., large] = 0, 0
    k[:, 7] = 0
    big_q, big_k = q.copy(), k.copy()
    big_q[..., large] = 2.0 ** 46
    big_k[:, 7, :, :32][..., large[:32]] = sign * 1.25 * 2.0 ** 45
    big_k[:, 7, :, 32:64][..., large[32:64]] = -sign * 1.25 * 2.0 ** 45
    assert ordinary.any()
    A = D.Array.from_numpy
    check_forward(D, q, k, v, counts, np.log(2.0), D.op.cross_attention(A(big_q), A(big_k), A(v), A(counts), np.log(2.0)))
    # smaller ordinary scores, so that the state weighs as much as others do whatever the width
    for a in (q, big_q):
        a[..., ordinary] *= np.float32(4.0 / width)
    check_forward(D, q, k, v, counts, np.log(2.0), D.op.cross_attention(A(big_q), A(big_k), A(v), A(counts), np.log(2.0)))


@pytest.mark.parametrize("queries", [1, 12, 70])
@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("keys", [1, 15, 33, 90, 700])
def test_an_infinite_value_of_the_last_state(gpu, D, rng, queries, dtype, keys):
    """It comes out in its own column, whatever the kernel puts in the places behind the last state."""
    A, op = D.Array.from_numpy, D.op
    for width in (8, 64, 128, 256):
        q, k, v, _ = make(rng, dtype, 2, queries, keys, 2, 1, width)
        counts = np.array([keys, max(1, keys - 9)], np.int32)
        for b in range(2):
            v[b, counts[b] - 1, 0, 3] = np.inf
        y, lse = (a.numpy() for a in op.cross_attention(A(q), A(k), A(v), A(counts), 0.1))
        assert np.isfinite(lse).all() and (y[..., 3] == np.inf).all()
        clean = v.copy()
        clean[..., 3], y[..., 3] = 0, 0
        check_forward(D, q, k, clean, counts, 0.1, (A(y), A(lse)))


@pytest.mark.parametrize("width", [32, 64, 128, 256])
def test_gradients_with_a_small_scale(gpu, D, rng, width):
    """A scale of 1e-33, whose gradients dy of about 2^60 brings back to ordinary numbers."""
    q, k, v, counts = make(rng, np.float32, 2, 70, 90, 2, 1, width, [90, 47])
    check_backward(D, (rng.randn(*q.shape) * 2.0 ** 60).astype(np.float32), q, k, v, counts, 1e-33)


@pytest.mark.parametrize("width", [129, 160, 187, 192, 193, 256])
@pytest.mark.parametrize("queries,keys", [(40, 90), (19, 333)])
def test_wide_heads_in_double_precision(gpu, D, rng, width, queries, keys):
    """Two waves to a row: padded batches, views, destinations between other values, recordings."""
    A, op = D.Array.from_numpy, D.op
    q, k, v, counts = make(rng, np.float64, 4, queries, keys, 4, 2, width, [0, 1, keys, 33])
    dy = rng.randn(*q.shape)
    behind = np.arange(keys)[None, :] >= counts[:, None]
    k[behind], v[behind] = np.nan, np.inf
    scale = 1 / np.sqrt(width)
    y, lse = check_forward(D, q, k, v, counts, scale)
    grads = check_backward(D, dy, q, k, v, counts, scale)
    turned = lambda a: A(np.ascontiguousarray(a.transpose(0, 2, 1, 3))).transpose(0, 2, 1, 3)  # noqa: E731
    wider = A(np.concatenate([v, k, np.full(k.shape[:3] + (1,), np.nan)], 3))
    views = (A(q[:, ::-1].copy())[:, ::-1], wider[:, :, :, width:2 * width], turned(v))
    for a, b in zip((y, lse), op.cross_attention(*views, A(counts), scale)):
        assert np.array_equal(a.numpy(), b.numpy())
    for a, b in zip(grads, op.cross_attention_backward(turned(dy), *views, y, lse, A(counts), scale)):
        assert np.array_equal(a.numpy(), b.numpy())
    # destinations inside longer arrays: what lies before and behind stays
    longer = [A(np.full((6,) + s[1:], 7.0)) for s in (q.shape, q.shape[:3], q.shape, k.shape, k.shape)]
    inside = [a[1:5] for a in longer]
    ins = [A(a) for a in (dy, q, k, v, counts)]
    rec = D.Recording()
    with rec:
        op.cross_attention(*ins[1:], scale, out=inside[:2])
        op.cross_attention_backward(*ins[:4], *inside[:2], ins[4], scale, out=inside[2:])
    rec.make_graph()
    for _ in range(3):
        for a in inside:
            a.assign(a * 0.0)
        op.cross_attention(ins[1] * 2.0, ins[2], ins[3], ins[4])[0].numpy()  # the program's own work in between
        rec.replay()
        for got, want in zip(longer, (y, lse) + tuple(grads)):
            assert (got.numpy()[[0, 5]] == 7).all() and np.array_equal(got.numpy()[1:5], want.numpy())

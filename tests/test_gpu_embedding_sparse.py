"""The gradient of an embedding table most of whose rows no token names (from 16384 rows on zeros go over many of them at once), against the formula in 64 bits and more."""
import numpy as np
import pytest

from test_gpu_embedding import check_gradient, tokens_of

pytestmark = pytest.mark.gpu

# rows, width, tokens: around a row of one group, 32 groups, 64 groups; short rows with nearly as many tokens as rows; a row of more than 32 KiB; fewer rows,
# of more than 256 MiB
SIZES = [(16384, 1, 300), (16384, 3, 16000), (20011, 4, 900), (20000, 5, 19000), (16400, 33, 1000), (17000, 64, 40), (16500, 65, 1000), (16384, 129, 900), (16391, 131, 1), (20000, 257, 500),
         (16384, 513, 300), (16500, 1030, 200), (16384, 8200, 20), (8000, 8500, 20)]


def near_and_far(rng, count, rows):
    """Tokens of every kind: heavy ones, whose runs lie in several parts, the first and last row, neighbours, and outside."""
    tokens = tokens_of(rng, count, rows)
    if count >= 20:
        tokens[: count // 3] = rows // 2
        tokens[-6:] = [0, rows - 1, rows - 1, 7, 8, rows]
    return tokens[rng.permutation(count)]


@pytest.mark.parametrize("rows,width,count", SIZES)
@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_gradient(gpu, D, rng, rows, width, count, dtype):
    if width > 8192 and dtype == np.float64:
        width //= 2
    dy, tokens = rng.randn(count, width).astype(dtype), near_and_far(rng, count, rows)
    out = D.Array.from_numpy(np.full((rows, width), np.nan, dtype))
    D.op.embedding_backward(D.Array.from_numpy(dy), D.Array.from_numpy(tokens), rows, 1.5, out=out)
    check_gradient(out.numpy(), dy, tokens, rows, 1.5)


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_a_destination_off_16_bytes_between_others(gpu, D, rng, dtype):
    """Rows inside a longer array, which begin anywhere: what lies before and behind stays."""
    for first, width in ((1, 5), (3, 33), (2, 131)):
        rows, count = 16390, 500
        dy, tokens = rng.randn(count, width).astype(dtype), near_and_far(rng, count, rows)
        whole = D.Array.from_numpy(np.full((first + rows + 2, width), 7.0, dtype))
        D.op.embedding_backward(D.Array.from_numpy(dy), D.Array.from_numpy(tokens), rows, out=whole[first:first + rows])
        got = whole.numpy()
        assert (got[:first] == 7).all() and (got[first + rows:] == 7).all()
        check_gradient(got[first:first + rows], dy, tokens, rows, 1.0)


def test_no_token_inside(gpu, D):
    for width in (6, 300):
        for count in (0, 40):
            got = D.op.embedding_backward(D.Array.from_numpy(np.full((count, width), np.nan, np.float32)) if count else D.Array.empty((0, width)),
                                          D.Array.from_numpy(np.full(count, -1, np.int32)) if count else D.Array.empty((0,), D.DTYPE_INT32), 17001)
            assert got.shape == (17001, width) and (got.numpy() == 0).all()


def test_recorded_and_replayed(gpu, D, rng):
    op = D.op
    rows, count, width = 16401, 700, 50
    tokens, dy = D.Array.from_numpy(near_and_far(rng, count, rows)), D.Array.from_numpy(rng.randn(count, width).astype(np.float32))
    dtable = D.Array.empty((rows, width))
    rec = D.Recording()
    with rec:
        op.embedding_backward(dy, tokens, rows, 0.5, out=dtable)
    rec.make_graph()
    for _ in range(3):
        other = near_and_far(rng, count, rows)
        tokens.assign(D.Array.from_numpy(other))
        dy.assign(dy * -0.5)
        dtable.assign(dtable * 0.0 + 1.0)
        op.embedding_backward(dy * 1.0, D.Array.from_numpy(other[::-1].copy()), rows).numpy()  # the program's own work in between
        rec.replay()
        check_gradient(dtable.numpy(), dy.numpy(), other, rows, 0.5)

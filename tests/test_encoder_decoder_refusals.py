"""What embedding rows, cross attention and the cross entropy of a projection refuse before they touch a device: types, shapes, counts and destinations."""
import ctypes as C

import numpy as np
import pytest


def test_embedding(D):
    op, E = D.op, D.Array.empty
    table, tokens, y = E((7, 4)), E((5,), D.DTYPE_INT32), E((5, 4))
    for call, text in ((lambda: op.embedding(E((7, 4), D.DTYPE_INT32), tokens), "float or double matrix"), (lambda: op.embedding(E((7,)), tokens), "matrix"),
                       (lambda: op.embedding(E((0, 4)), tokens), "not empty"), (lambda: op.embedding(table, E((5,))), "tokens must be int"),
                       (lambda: op.embedding(table, tokens, float("inf")), "scale must be finite"), (lambda: op.embedding(table, tokens, 1.0, out=E((4, 5))), "y must be"),
                       (lambda: op.embedding(table, tokens, 1.0, out=E((4, 5)).T), "dense buffer"), (lambda: op.embedding(table, tokens, 1.0, out=E((5, 4), D.DTYPE_DOUBLE)), "y must be float"),
                       (lambda: op.embedding_backward(y, E((4,), D.DTYPE_INT32), 7), "tokens must be"), (lambda: op.embedding_backward(y, E((5,)), 7), "tokens must be"),
                       (lambda: op.embedding_backward(y, tokens, 0), "at least one row"), (lambda: op.embedding_backward(y, tokens, 2 ** 40), "at least one row"),
                       (lambda: op.embedding_backward(y, tokens, -3), "at least one row"), (lambda: op.embedding_backward(y, tokens, 7, float("nan")), "scale must be finite"),
                       (lambda: op.embedding_backward(E((5, 0)), tokens, 7), "last axis"), (lambda: op.embedding_backward(y, tokens, 7, out=E((6, 4))), "dtable must be")):
        with pytest.raises(D.DaliError, match=text):
            call()
    with pytest.raises((TypeError, ValueError)):
        op.embedding(table, tokens, "one")
    with pytest.raises(TypeError):
        op.embedding_backward(y, tokens, "seven")


def test_cross_attention(D):
    op, E = D.op, D.Array.empty
    q, k, counts = E((2, 5, 6, 8)), E((2, 9, 3, 8)), E((2,), D.DTYPE_INT32)
    lse = E((2, 5, 6))
    calls = [(lambda: op.cross_attention(E((2, 5, 6)), k, k), "queries must be"), (lambda: op.cross_attention(E((2, 5, 6, 8), D.DTYPE_INT32), k, k), "queries must be"),
             (lambda: op.cross_attention(q, E((2, 9, 3, 7)), k), "keys must be"), (lambda: op.cross_attention(q, E((3, 9, 3, 8)), k), "keys must be"),
             (lambda: op.cross_attention(q, E((2, 9, 3, 8), D.DTYPE_DOUBLE), k), "keys must be"), (lambda: op.cross_attention(q, k, E((2, 8, 3, 8))), "values must be"),
             (lambda: op.cross_attention(q, E((2, 9, 4, 8)), E((2, 9, 4, 8))), "6 heads cannot share 4"), (lambda: op.cross_attention(q, k, k, E((3,), D.DTYPE_INT32)), "key_counts must be"),
             (lambda: op.cross_attention(q, k, k, E((2,))), "key_counts must be int"), (lambda: op.cross_attention(q, k, k, counts, float("nan")), "scale must be finite"),
             (lambda: op.cross_attention(E((1, 1, 1, 257)), E((1, 1, 1, 257)), E((1, 1, 1, 257))), "1 to 256 wide"),
             (lambda: op.cross_attention(q, k, k, out=(lse, None)), "y must be"), (lambda: op.cross_attention(q, k, k, out=(None, q)), "lse must be"),
             (lambda: op.cross_attention_backward(k, q, k, k, q, lse), "dy must be"), (lambda: op.cross_attention_backward(q, q, k, k, k, lse), "y must be"),
             (lambda: op.cross_attention_backward(q, q, k, k, q, q), "lse must be"), (lambda: op.cross_attention_backward(q, q, k, k, q, lse, out=(k, None, None)), "d_queries must be"),
             (lambda: op.cross_attention_backward(q, q, k, k, q, lse, out=(None, q, None)), "d_keys must be"),
             (lambda: op.cross_attention_backward(q, q, k, k, q, lse, out=(None, None, q)), "d_values must be")]
    for call, text in calls:
        with pytest.raises(D.DaliError, match=text):
            call()
    with pytest.raises(TypeError, match="out must hold 2"):
        op.cross_attention(q, k, k, out=(None,))
    with pytest.raises(TypeError, match="out must hold 3"):
        op.cross_attention_backward(q, q, k, k, q, lse, out=(None, None))


def test_projected_cross_entropy(D):
    op, E = D.op, D.Array.empty
    x, w, targets, bias, per_row = E((4, 6)), E((6, 9)), E((4,), D.DTYPE_INT32), E((9,)), E((4,))
    for call, text in ((lambda: op.projected_cross_entropy(E((4, 6), D.DTYPE_INT32), w, targets), "x must be"), (lambda: op.projected_cross_entropy(E((4, 0)), w, targets), "last axis"),
                       (lambda: op.projected_cross_entropy(x, E((5, 9)), targets), "w must be float"), (lambda: op.projected_cross_entropy(x, E((6, 0)), targets), "w must be"),
                       (lambda: op.projected_cross_entropy(x, E((6, 9), D.DTYPE_DOUBLE), targets), "w must be float"), (lambda: op.projected_cross_entropy(x, w, per_row), "targets must be int"),
                       (lambda: op.projected_cross_entropy(x, w, E((5,), D.DTYPE_INT32)), "targets must be"), (lambda: op.projected_cross_entropy(x, w, targets, per_row), "bias must be"),
                       (lambda: op.projected_cross_entropy(x, w, targets, out=(bias, None)), "losses must be"), (lambda: op.projected_cross_entropy(x, w, targets, out=(None, bias)), "lse must be"),
                       (lambda: op.projected_cross_entropy_backward(bias, x, w, targets, per_row), "d_losses must be"),
                       (lambda: op.projected_cross_entropy_backward(per_row, x, w, targets, bias), "lse must be"),
                       (lambda: op.projected_cross_entropy_backward(per_row, x, w, targets, per_row, out=(None, None, bias)), "without bias"),
                       (lambda: op.projected_cross_entropy_backward(per_row, x, w, targets, per_row, out=(w, None, None)), "dx must be"),
                       (lambda: op.projected_cross_entropy_backward(per_row, x, w, targets, per_row, out=(None, E((9, 6)), None)), "dw must be"),
                       (lambda: op.projected_cross_entropy_backward(per_row, x, w, targets, per_row, bias, out=(None, None, per_row)), "dbias must be")):
        with pytest.raises(D.DaliError, match=text):
            call()


def test_entries_of_the_library(D):
    """The C entries say what is wrong with their arguments and launch nothing (no device is needed to hear it)."""
    from dali_amd._native import hip
    host = (C.c_double * 4096)()
    base = (C.addressof(host) + 255) // 256 * 256
    p = [C.c_void_p(base + 2048 * i) for i in range(12)]
    size = C.c_size_t()

    def refused(status, text):
        assert status != 0 and text in hip.dali_hip_last_error().decode(), hip.dali_hip_last_error()

    refused(hip.dali_hip_embedding(9, 4, 5, 6, p[0], 6, p[1], 1.0, p[2]), "dtype")
    refused(hip.dali_hip_embedding(0, -1, 5, 6, p[0], 6, p[1], 1.0, p[2]), "tokens")
    refused(hip.dali_hip_embedding(0, 4, 0, 6, p[0], 6, p[1], 1.0, p[2]), "table of 0 rows")
    refused(hip.dali_hip_embedding(0, 4, 5, 0, p[0], 6, p[1], 1.0, p[2]), "rows of 0 values")
    refused(hip.dali_hip_embedding(0, 4, 5, 6, p[0], 6, p[1], float("nan"), p[2]), "finite")
    refused(hip.dali_hip_embedding(0, 4, 5, 6, None, 6, p[1], 1.0, p[2]), "NULL")
    refused(hip.dali_hip_embedding(0, 4, 5, 6, C.c_void_p(base + 2), 6, p[1], 1.0, p[2]), "off its type")
    refused(hip.dali_hip_embedding(0, 4, 5, 6, p[0], 6, p[1], 1.0, C.c_void_p(base + 64)), "overlaps")
    refused(hip.dali_hip_embedding_backward(0, 4, 5, 6, p[0], 6, p[1], 1.0, p[2], None), "NULL")
    refused(hip.dali_hip_embedding_backward(0, 4, 5, 6, p[0], 6, p[1], 1.0, p[2], C.c_void_p(base + 8192 + 16)), "256 bytes")
    refused(hip.dali_hip_embedding_backward_workspace(0, 2 ** 33, 5, 6, C.byref(size)), "tokens")

    strides = (C.c_int64 * 3)(64, 16, 8)
    sizes = (0, 1, 4, 4, 2, 1, 8)
    forward = lambda z, q=p[0], y=p[3], lse=p[4], space=p[5]: hip.dali_hip_cross_attention(*z, q, strides, p[1], strides, p[2], strides, None, 1.0, y, lse, space)  # noqa: E731
    refused(forward((7,) + sizes[1:]), "dtype")
    refused(forward((0, -1) + sizes[2:]), "sequences")
    refused(forward((0, 1, 4, 4, 3, 2, 8)), "3 heads cannot share 2")
    refused(forward((0, 1, 4, 4, 2, 1, 257)), "256 wide")
    refused(forward((0, 2 ** 20, 2 ** 27, 4, 8, 1, 8)), "too many")
    refused(forward(sizes, q=None), "NULL")
    refused(forward(sizes, y=C.c_void_p(base + 1)), "off its type")
    refused(forward(sizes, y=p[0]), "overlaps")
    refused(hip.dali_hip_cross_attention_backward(*sizes, p[6], strides, p[0], strides, p[1], strides, p[2], strides, p[3], None, None, 1.0, p[7], p[8], p[9], p[10]), "NULL")
    refused(hip.dali_hip_cross_attention_backward(*sizes, p[6], strides, p[0], strides, p[1], strides, p[2], strides, p[3], p[4], None, 1.0, p[7], p[8], p[8], p[10]), "overlap")
    refused(hip.dali_hip_cross_attention_workspace(*sizes, 0, None), "NULL")

    refused(hip.dali_hip_projected_cross_entropy(0, 4, 0, 9, p[0], 6, p[1], 9, 0, None, p[2], p[3], p[4], p[5]), "rows of 0 values")
    refused(hip.dali_hip_projected_cross_entropy(0, 4, 6, 0, p[0], 6, p[1], 9, 0, None, p[2], p[3], p[4], p[5]), "vocabulary of 0")
    refused(hip.dali_hip_projected_cross_entropy(0, 4, 6, 9, p[0], 5, p[1], 9, 0, None, p[2], p[3], p[4], p[5]), "values apart")
    refused(hip.dali_hip_projected_cross_entropy(0, 4, 6, 9, p[0], 6, p[1], 8, 0, None, p[2], p[3], p[4], p[5]), "w's stride")
    refused(hip.dali_hip_projected_cross_entropy(0, 4, 6, 9, p[0], 6, p[1], 5, 1, None, p[2], p[3], p[4], p[5]), "w's stride")
    refused(hip.dali_hip_projected_cross_entropy(0, 4, 6, 9, p[0], 6, p[1], 9, 0, None, p[2], p[3], p[3], p[5]), "overlap")
    refused(hip.dali_hip_projected_cross_entropy_backward(0, 4, 6, 9, p[0], p[1], 6, p[2], 9, 0, None, p[3], p[4], p[5], p[6], 0, p[7], p[8]), "come together")
    for z in ((0, 700, 32, 9000, 0, 0), (0, 700, 32, 9000, 1, 1), (1, 700, 32, 9000, 1, 1), (0, 3, 32, 90, 0, 0), (0, 0, 32, 90, 1, 0)):
        assert hip.dali_hip_projected_cross_entropy_workspace(*z, C.byref(size)) == 0
        assert (size.value > 0) == (z[1] > 0)

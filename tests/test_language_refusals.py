"""What the operators of language models refuse before they touch a device: types, shapes, counts and destinations."""
import ctypes as C

import numpy as np
import pytest


def arrays(D):
    A = D.Array.from_numpy
    return (A(np.zeros((4, 6), np.float32)), A(np.zeros((4,), np.float32)), A(np.zeros((6,), np.float32)), A(np.zeros((4,), np.int32)), A(np.zeros((4, 6))), A(np.zeros((4, 6), np.int32)))


def test_layer_norm(D):
    op = D.op
    x, per_row, vector, tokens, double, whole = arrays(D)
    for call, text in ((lambda: op.layer_norm(whole), "float or double"), (lambda: op.layer_norm(D.Array.empty(())), "last axis"), (lambda: op.layer_norm(D.Array.empty((3, 0))), "last axis"),
                       (lambda: op.layer_norm(x, per_row), "gamma must be float of shape"), (lambda: op.layer_norm(x, vector, per_row), "beta must be float of shape"),
                       (lambda: op.layer_norm(double, vector), "gamma must be double"), (lambda: op.layer_norm(x, x), "gamma must be"),
                       (lambda: op.layer_norm(x, out=(double, None, None)), "y must be float"), (lambda: op.layer_norm(x, out=(None, vector, None)), "mean must be"),
                       (lambda: op.layer_norm(x, out=(D.Array.empty((6, 4)).T, None, None)), "dense buffer"), (lambda: op.layer_norm(x, out=(x + 1.0, None, None)), "dense buffer"),
                       (lambda: op.layer_norm_backward(x, x, vector, per_row), "mean must be"), (lambda: op.layer_norm_backward(x, x, per_row, vector), "rstd must be"),
                       (lambda: op.layer_norm_backward(double, x, per_row, per_row), "dy must be"), (lambda: op.layer_norm_backward(x.T, x, per_row, per_row), "dy must be"),
                       (lambda: op.layer_norm_backward(x, x, per_row, per_row, per_row), "gamma must be"),
                       (lambda: op.layer_norm_backward(x, x, per_row, per_row, out=(None, vector, None)), "without gamma"),
                       (lambda: op.layer_norm_backward(x, x, per_row, per_row, vector, out=(None, None, per_row)), "dbeta must be")):
        with pytest.raises(D.DaliError, match=text):
            call()
    with pytest.raises(TypeError):
        op.layer_norm(x, epsilon="small")
    with pytest.raises(TypeError, match="out must hold 3"):
        op.layer_norm(x, out=(x,))
    with pytest.raises(TypeError, match="no Array"):
        op.layer_norm(x, out=(np.zeros((4, 6), np.float32), None, None))


def test_token_log_probs(D):
    op = D.op
    x, per_row, vector, tokens, double, whole = arrays(D)
    for call, text in ((lambda: op.token_log_probs(whole, tokens), "float or double"), (lambda: op.token_log_probs(x, per_row), "tokens must be int"),
                       (lambda: op.token_log_probs(x, whole), "tokens must be int"), (lambda: op.token_log_probs(x, tokens, -1), "k must be from 0 to 6"),
                       (lambda: op.token_log_probs(x, tokens, 7), "k must be from 0 to 6"), (lambda: op.token_log_probs(D.Array.empty((4, 900)), tokens, 65), "k must be from 0 to 64"),
                       (lambda: op.token_log_probs(x, tokens, 2 ** 32 + 1), "k must be from 0 to 6"), (lambda: op.token_log_probs(x, tokens, 10 ** 30), "k must be from 0 to 6"),
                       (lambda: op.token_log_probs(D.Array.empty((4, 0)), tokens), "last axis"),
                       (lambda: op.token_log_probs(x, tokens, 0, out=(None, None, None, x, None)), "with k = 0"), (lambda: op.token_log_probs(x, tokens, 2, out=(None, None, None, x, None)), "top_log_probs must be"),
                       (lambda: op.token_log_probs(x, tokens, 2, out=(None, None, None, None, D.Array.empty((4, 2)))), "top_tokens must be int"),
                       (lambda: op.token_log_probs_backward(vector, None, x, tokens, per_row, None), "d_log_probs must be"),
                       (lambda: op.token_log_probs_backward(per_row, per_row, x, tokens, per_row, None), "needs the entropy"),
                       (lambda: op.token_log_probs_backward(per_row, vector, x, tokens, per_row, per_row), "d_entropy must be"),
                       (lambda: op.token_log_probs_backward(per_row, None, x, tokens, vector, None), "lse must be"),
                       (lambda: op.token_log_probs_backward(per_row, None, x, tokens, per_row, None, out=double), "d_logits must be")):
        with pytest.raises(D.DaliError, match=text):
            call()
    with pytest.raises(TypeError, match="out must hold 5"):
        op.token_log_probs(x, tokens, 0, out=(None, None))


def test_clip_by_global_norm(D):
    op = D.op
    x, per_row, vector, tokens, double, whole = arrays(D)
    for call, text in ((lambda: op.clip_by_global_norm([], 1.0), "at least one"), (lambda: op.global_norm([]), "at least one"), (lambda: op.global_norm([tokens]), "all of one type"),
                       (lambda: op.clip_by_global_norm([x, double], 1.0), "all of one type"), (lambda: op.clip_by_global_norm([x], -1.0), "must not be negative"),
                       (lambda: op.clip_by_global_norm([x], float("nan")), "must not be negative"), (lambda: op.clip_by_global_norm([x], 1.0, out=([vector], None)), "an array must be"),
                       (lambda: op.clip_by_global_norm([x], 1.0, out=([D.Array.empty((6, 4)).T], None)), "dense buffer"),
                       (lambda: op.clip_by_global_norm([x], 1.0, out=(None, vector)), "the norm must be float of shape")):
        with pytest.raises(D.DaliError, match=text):
            call()
    with pytest.raises(TypeError, match="out must hold 2"):
        op.clip_by_global_norm([x, x], 1.0, out=([x], None))
    with pytest.raises((TypeError, ValueError)):
        op.clip_by_global_norm([x], "one")


def test_entries_of_the_library(D):
    """The C entries say what is wrong with their arguments and launch nothing (no device is needed to hear it)."""
    from dali_amd._native import hip
    host = (C.c_double * 64)()
    p = C.cast(host, C.c_void_p)

    def refused(status, text):
        assert status != 0 and text in hip.dali_hip_last_error().decode(), hip.dali_hip_last_error()

    at = lambda i: C.c_void_p(C.addressof(host) + 8 * i)  # noqa: E731
    refused(hip.dali_hip_layer_norm(2, 1, 4, p, 4, None, None, 1e-5, p, p, p), "neither float nor double")
    refused(hip.dali_hip_layer_norm(0, -1, 4, p, 4, None, None, 1e-5, p, p, p), "-1 rows")
    refused(hip.dali_hip_layer_norm(0, 1, 0, p, 4, None, None, 1e-5, p, p, p), "0 values")
    refused(hip.dali_hip_layer_norm(0, 1, 4, None, 4, None, None, 1e-5, p, p, p), "NULL")
    refused(hip.dali_hip_layer_norm(0, 1, 4, p, 4, None, None, -1.0, at(8), at(16), at(17)), "epsilon")
    refused(hip.dali_hip_layer_norm(1, 1, 4, p, 4, None, None, 1e-5, at(2), at(16), at(17)), "y overlaps x")
    refused(hip.dali_hip_layer_norm(1, 2, 4, at(4), -4, None, None, 1e-5, p, at(16), at(20)), "y overlaps x")  # (rows that run backwards reach below their start)
    refused(hip.dali_hip_layer_norm_backward(1, 1, 4, p, 4, at(8), 4, at(16), at(17), at(20), at(24), at(28), None), "come together")
    refused(hip.dali_hip_layer_norm_backward(1, 1, 4, p, 4, at(8), 4, at(16), at(17), at(20), at(24), at(28), at(28)), "dgamma and dbeta overlap")
    refused(hip.dali_hip_token_log_probs(0, 1, 4, p, 4, p, 5, p, p, p, p, p), "5 alternatives")
    refused(hip.dali_hip_token_log_probs(0, 1, 400, p, 4, p, 65, p, p, p, p, p), "65 alternatives")
    refused(hip.dali_hip_token_log_probs(0, 1, 4, p, 4, p, 2, at(8), at(9), at(10), None, None), "NULL")
    refused(hip.dali_hip_token_log_probs_backward(0, 1, 4, p, p, p, 4, p, p, None, p), "NULL")
    odd = lambda i: C.c_void_p(C.addressof(host) + 8 * i + 2)  # noqa: E731
    refused(hip.dali_hip_layer_norm(0, 1, 4, odd(0), 4, None, None, 1e-5, at(8), at(16), at(17)), "off its type's size")
    refused(hip.dali_hip_layer_norm_backward(0, 1, 4, at(0), 4, at(8), 4, at(16), at(17), at(20), odd(24), at(28), at(32)), "off its type's size")
    refused(hip.dali_hip_token_log_probs(0, 1, 4, at(0), 4, odd(8), 0, at(10), at(11), at(12), None, None), "off its type's size")
    refused(hip.dali_hip_token_log_probs_backward(0, 1, 4, at(6), None, at(0), 4, at(8), at(9), None, odd(10)), "off its type's size")
    refused(hip.dali_hip_clip_by_global_norm(0, 1, (C.c_void_p * 1)(odd(0).value), None, (C.c_int64 * 1)(3), 1.0, at(9)), "off its type's size")
    sizes, pointers = (C.c_int64 * 1)(-3), (C.c_void_p * 1)(C.addressof(host))
    refused(hip.dali_hip_clip_by_global_norm(0, 1, pointers, None, sizes, 1.0, at(9)), "negative size")
    refused(hip.dali_hip_clip_by_global_norm(0, 1, pointers, pointers, (C.c_int64 * 1)(3), float("nan"), at(9)), "negative")
    refused(hip.dali_hip_clip_by_global_norm(0, 1, pointers, None, (C.c_int64 * 1)(3), 1.0, None), "NULL")
    assert hip.dali_hip_layer_norm(0, 0, 4, None, 4, None, None, 1e-5, None, None, None) == 0  # nothing to do
    assert hip.dali_hip_token_log_probs(0, 0, 4, None, 4, None, 0, None, None, None, None, None) == 0


def test_operands_without_a_handle(D):
    """An array whose handle was given up is no absent weight."""
    op = D.op
    x, per_row, vector, tokens, double, whole = arrays(D)
    gone = D.Array.from_numpy(np.zeros(6, np.float32))
    handle, gone._h = gone._h, None
    try:
        for call in (lambda: op.layer_norm(x, gone), lambda: op.layer_norm(x, vector, gone), lambda: op.layer_norm_backward(x, x, per_row, per_row, gone),
                     lambda: op.token_log_probs_backward(per_row, gone, x, tokens, per_row, None), lambda: op.token_log_probs_backward(per_row, per_row, x, tokens, per_row, gone)):
            with pytest.raises(TypeError, match="without a handle"):
                call()
        with pytest.raises(D.DaliError, match="NULL array handle"):
            op.layer_norm(gone)
    finally:
        gone._h = handle


@pytest.mark.parametrize("epsilon", [-1e-5, -np.inf, np.nan, 2e30, np.inf])
def test_epsilon(D, epsilon):
    from dali_amd._native import hip
    host = (C.c_double * 64)()
    at = lambda i: C.c_void_p(C.addressof(host) + 8 * i)  # noqa: E731
    for dtype in (0, 1):
        assert hip.dali_hip_layer_norm(dtype, 1, 4, at(0), 4, None, None, epsilon, at(8), at(16), at(17)) != 0
        assert "epsilon must be from 0 to 1e30" in hip.dali_hip_last_error().decode()

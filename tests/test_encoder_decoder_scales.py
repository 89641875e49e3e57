"""Scales that are finite in double and not in the operands' type are refused: as a factor in fp32 they are infinite, and times 0 NaN."""
import ctypes as C

import pytest


def test_front_end(D):
    op, E = D.op, D.Array.empty
    table, tokens, y = E((7, 4)), E((5,), D.DTYPE_INT32), E((5, 4))
    q, k, lse = E((2, 5, 6, 8)), E((2, 9, 3, 8)), E((2, 5, 6))
    for scale in (1e39, -1e300):
        for call in (lambda: op.embedding(table, tokens, scale), lambda: op.embedding_backward(y, tokens, 7, scale), lambda: op.cross_attention(q, k, k, None, scale),
                     lambda: op.cross_attention_backward(q, q, k, k, q, lse, None, scale)):
            with pytest.raises(D.DaliError, match="scale must be finite"):
                call()


def test_entries_of_the_library(D):
    from dali_amd._native import hip
    host = (C.c_double * 8192)()
    base = (C.addressof(host) + 255) // 256 * 256
    p = [C.c_void_p(base + 4096 * i) for i in range(12)]

    def refused(status):
        assert status != 0 and "scale must be finite" in hip.dali_hip_last_error().decode(), hip.dali_hip_last_error()

    strides = (C.c_int64 * 3)(64, 16, 8)
    sizes = (1, 4, 4, 2, 1, 8)
    for scale in (1e39, -1e300):
        refused(hip.dali_hip_embedding(0, 4, 5, 6, p[0], 6, p[1], scale, p[2]))
        refused(hip.dali_hip_embedding_backward(0, 4, 5, 6, p[0], 6, p[1], scale, p[2], p[3]))
    # (attention in fp32 counts its exponents in powers of two: log2 e more)
    for scale in (1e39, -3e38, 2.4e38):
        refused(hip.dali_hip_cross_attention(0, *sizes, p[0], strides, p[1], strides, p[2], strides, None, scale, p[3], p[4], p[5]))
        refused(hip.dali_hip_cross_attention_backward(0, *sizes, p[6], strides, p[0], strides, p[1], strides, p[2], strides, p[3], p[4], None, scale, p[7], p[8], p[9], p[10]))
    for dtype, scale in ((0, 2.3e38), (1, 1e300)):
        # (refused for another reason, behind the scale)
        assert hip.dali_hip_cross_attention(dtype, *sizes, None, strides, p[1], strides, p[2], strides, None, scale, p[3], p[4], p[5]) != 0
        assert "NULL" in hip.dali_hip_last_error().decode()

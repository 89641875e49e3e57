"""Operators of language models over more rows than one launch takes: what lies behind the end of the first launch against the same rows among few, bit for bit."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

ROWS = (1 << 23) + 5  # a launch takes 2^23 workgroups, and as many rows


def call(name, *args):
    from dali_amd._native import hip, hip_check
    hip_check(getattr(hip, name)(*args), name)


def ptr(array):
    return C.c_void_p(array.device_ptr())


def pattern(rng, rows, vocab):
    """Rows that repeat after `rows`, and what belongs to them"""
    return (rng.randn(rows, vocab) * 3).astype(np.float32), rng.randint(-1, vocab, rows).astype(np.int32), rng.randn(rows).astype(np.float32), rng.randn(rows).astype(np.float32)


def test_short_rows(gpu, D, rng):
    op, A, period, vocab, k = D.op, D.Array.from_numpy, 1021, 8, 3
    x, tokens, g, h = pattern(rng, period, vocab)
    which = np.arange(ROWS) % period
    small = [A(v) for v in (x, tokens, g, h)]
    large = [A(v[which]) for v in (x, tokens, g, h)]
    want, got = op.token_log_probs(small[0], small[1], k), op.token_log_probs(large[0], large[1], k)
    for p, q in zip(got, want):
        assert np.array_equal(p.numpy(), q.numpy()[which])
    d = op.token_log_probs_backward(small[2], small[3], small[0], small[1], want[2], want[1]).numpy()
    assert np.array_equal(op.token_log_probs_backward(large[2], large[3], large[0], large[1], got[2], got[1]).numpy(), d[which])


@pytest.mark.parametrize("k", [0, 4])
def test_long_rows(gpu, D, rng, k):
    """One row of logits for all (a stride of 0), another token for each."""
    op, A, vocab, few = D.op, D.Array.from_numpy, 2049, 2049
    x = (rng.randn(1, vocab) * 3).astype(np.float32)
    tokens = np.arange(ROWS, dtype=np.int32) % vocab
    row = A(x)
    outs = [D.Array.empty((ROWS,)) for _ in range(3)] + ([D.Array.empty((ROWS, k)), D.Array.empty((ROWS, k), D.DTYPE_INT32)] if k else [])
    t = A(tokens)
    call("dali_hip_token_log_probs", 0, ROWS, vocab, ptr(row), 0, ptr(t), k, *([ptr(o) for o in outs] + [None] * (5 - len(outs))))
    want = op.token_log_probs(A(np.repeat(x, few, 0)), A(tokens[:few]), k)
    for got, w in zip(outs, want):
        call("dali_hip_sync")
        buf = np.empty(got.shape, w.numpy().dtype)
        call("dali_hip_memcpy_d2h", buf.ctypes.data_as(C.c_void_p), ptr(got), buf.nbytes)
        assert np.array_equal(buf, w.numpy()[np.arange(ROWS) % few])


def test_gradient_of_long_rows(gpu, D, rng):
    op, A, vocab = D.op, D.Array.from_numpy, 1025
    x = (rng.randn(1, vocab) * 3).astype(np.float32)
    tokens = rng.randint(-1, vocab, ROWS).astype(np.int32)
    g, h = rng.randn(ROWS).astype(np.float32), rng.randn(ROWS).astype(np.float32)
    row = A(x)
    _, entropy, lse, _, _ = op.token_log_probs(row, A(tokens[:1]))
    e, l = np.repeat(entropy.numpy(), ROWS), np.repeat(lse.numpy(), ROWS)
    held = [A(v) for v in (g, h, tokens, l, e)]
    at = np.r_[0:3, (1 << 23) - 3:ROWS]
    want = op.token_log_probs_backward(A(g[at]), A(h[at]), A(np.repeat(x, len(at), 0)), A(tokens[at]), A(l[at]), A(e[at])).numpy()
    d = C.c_void_p()
    call("dali_hip_malloc", C.byref(d), 4 * ROWS * vocab)
    try:
        call("dali_hip_token_log_probs_backward", 0, ROWS, vocab, ptr(held[0]), ptr(held[1]), ptr(row), 0, ptr(held[2]), ptr(held[3]), ptr(held[4]), d)
        call("dali_hip_sync")
        got = np.empty((len(at), vocab), np.float32)
        for i, r in enumerate(at):
            call("dali_hip_memcpy_d2h", got[i].ctypes.data_as(C.c_void_p), C.c_void_p(d.value + 4 * vocab * int(r)), got[i].nbytes)
        assert np.array_equal(got, want)
    finally:
        call("dali_hip_free", d)

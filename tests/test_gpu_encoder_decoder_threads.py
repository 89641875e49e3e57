"""Two host threads that launch the operators of an encoder-decoder model at the same time: each gets what it gets alone, bit for bit."""
import ctypes as C
import threading

import numpy as np
import pytest

from test_gpu_language_threads import Call

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def made(D):
    from dali_amd._native import hip
    rng = np.random.RandomState(5)
    kept = []
    p = lambda a: C.c_void_p(a.device_ptr())  # noqa: E731

    def hold(a):
        kept.append(a)
        return p(a)

    # (matrices by the root of their rows, so that logits are of order one: weights e^90 would pass the type's range, and NaN is not equal to itself)
    new = lambda *s: hold(D.Array.from_numpy((rng.randn(*s) / (np.sqrt(s[0]) if len(s) == 2 else 1)).astype(np.float32)))  # noqa: E731
    tokens = lambda n, high: hold(D.Array.from_numpy(rng.randint(-1, high, n).astype(np.int32)))  # noqa: E731
    empty = D.Array.empty

    def space(entry, *extents):
        size = C.c_size_t()
        assert getattr(hip, entry)(*extents, C.byref(size)) == 0
        a = empty((size.value // 4 + 64,))
        kept.append(a)
        return C.c_void_p((a.device_ptr() + 255) // 256 * 256)

    def entropy_backward(rows, inputs, vocab):
        extents = (0, rows, inputs, vocab)
        d, x, w, b, lse, t, dw = new(rows), new(rows, inputs), new(inputs, vocab), new(vocab), new(rows), tokens(rows, vocab), hold(empty((inputs, vocab)))
        ws = space("dali_hip_projected_cross_entropy_workspace", *extents, 1, 1)
        return Call(D, "dali_hip_projected_cross_entropy_backward", [empty((rows, inputs)), empty((vocab,))],
                    lambda dx, db: (*extents, d, x, inputs, w, vocab, 0, b, t, lse, dx, dw, 0, db, ws))

    def entropy(rows, inputs, vocab):
        extents = (0, rows, inputs, vocab)
        x, w, t = new(rows, inputs), new(inputs, vocab), tokens(rows, vocab)
        ws = space("dali_hip_projected_cross_entropy_workspace", *extents, 0, 0)
        return Call(D, "dali_hip_projected_cross_entropy", [empty((rows,)), empty((rows,))], lambda losses, lse: (*extents, x, inputs, w, vocab, 0, None, t, losses, lse, ws))

    def attention(batch, keys, heads, width):
        extents = (0, batch, 1, keys, heads, 1, width)
        q, k, v = new(batch, heads, width), new(batch, keys, width), new(batch, keys, width)
        sq, sk = (C.c_int64 * 3)(heads * width, heads * width, width), (C.c_int64 * 3)(keys * width, width, width)
        kept.append((sq, sk))
        ws = space("dali_hip_cross_attention_workspace", *extents, 0)
        return Call(D, "dali_hip_cross_attention", [empty((batch, heads, width)), empty((batch, heads))], lambda y, lse: (*extents, q, sq, k, sk, v, sk, None, 0.1, y, lse, ws))

    def embedding_backward(count, rows, width):
        dy, t = new(count, width), tokens(count, rows)
        ws = space("dali_hip_embedding_backward_workspace", 0, count, rows, width)
        return Call(D, "dali_hip_embedding_backward", [empty((rows, width))], lambda dtable: (0, count, rows, width, dy, width, t, 1.0, dtable, ws))

    # (the gradients' products over 16000 and 9000 columns are cut into shares that another launch adds up)
    calls = {"gradients": entropy_backward(256, 512, 16000), "gradients again": entropy_backward(200, 384, 9000), "images": entropy_backward(600, 64, 7000), "few rows": entropy(5, 256, 9000),
             "positions": attention(3, 2000, 4, 64), "tokens": embedding_backward(5000, 300, 64), "many tokens": embedding_backward(30000, 300, 64)}
    yield calls
    del kept[:]


@pytest.mark.parametrize("first,second", [("gradients", "gradients again"), ("gradients", "images"), ("few rows", "positions"), ("gradients again", "tokens"), ("many tokens", "positions"),
                                          ("few rows", "few rows")])
def test_two_threads(gpu, D, made, first, second):
    failures = []
    names = [first] if first == second else [first, second]
    threads = [threading.Thread(target=made[name].repeat, args=(60, failures)) for name in names]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, failures[:5]

"""Two host threads that launch operators of language models at the same time: each gets what it gets alone, bit for bit."""
import ctypes as C
import threading

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


class Call(object):
    """An entry of the library with its operands, and the results that it gives alone"""

    def __init__(self, D, name, outs, arguments):
        from dali_amd._native import hip
        self.hip, self.name, self.outs = hip, name, outs
        self.pointers = [C.c_void_p(o.device_ptr()) for o in outs]
        self.arguments = arguments(*self.pointers)
        self.host = [np.empty(o.shape, np.float32) for o in outs]
        self.want = [v.copy() for v in self()]

    def __call__(self):
        status = getattr(self.hip, self.name)(*self.arguments)
        assert status == 0, self.hip.dali_hip_last_error()
        for p, h in zip(self.pointers, self.host):
            assert self.hip.dali_hip_memcpy_d2h(h.ctypes.data_as(C.c_void_p), p, h.nbytes) == 0
        return self.host

    def repeat(self, times, failures):
        try:
            for i in range(times):
                for k, (got, want) in enumerate(zip(self(), self.want)):
                    if not np.array_equal(got, want):
                        failures.append((self.name, i, k))
        except Exception as error:  # noqa: B902
            failures.append(error)


def calls(D, rng):
    new = lambda *s: D.Array.from_numpy(rng.randn(*s).astype(np.float32))  # noqa: E731
    p = lambda a: C.c_void_p(a.device_ptr())  # noqa: E731
    empty = D.Array.empty
    kept = []

    def hold(*arrays):
        kept.extend(arrays)
        return arrays if len(arrays) > 1 else arrays[0]

    def clip(n):
        grads = hold(*[new(n), new(77)])
        sizes, addresses = (C.c_int64 * 2)(n, 77), (C.c_void_p * 2)(*[g.device_ptr() for g in grads])
        return Call(D, "dali_hip_clip_by_global_norm", [empty((n,)), empty((77,)), empty(())],
                    lambda a, b, norm: (0, 2, addresses, (C.c_void_p * 2)(a.value, b.value), sizes, 1.0, norm))

    def norm_backward(rows, width):
        dy, x, mean, rstd, gamma = hold(new(rows, width), new(rows, width), new(rows), new(rows), new(width))
        return Call(D, "dali_hip_layer_norm_backward", [empty((rows, width)), empty((width,)), empty((width,))],
                    lambda dx, dg, db: (0, rows, width, p(dy), width, p(x), width, p(mean), p(rstd), p(gamma), dx, dg, db))

    def log_probs(rows, vocab):
        x, t = hold(new(rows, vocab), D.Array.from_numpy(rng.randint(0, vocab, rows).astype(np.int32)))
        return Call(D, "dali_hip_token_log_probs", [empty((rows,)), empty((rows,)), empty((rows,))], lambda a, b, c: (0, rows, vocab, p(x), vocab, p(t), 0, a, b, c, None, None))

    return kept, {"clip": clip(200000), "clip again": clip(150000), "norm_backward": norm_backward(700, 512), "norm_backward wide": norm_backward(70, 20000),
                  "log_probs": log_probs(3, 50257)}


@pytest.mark.parametrize("first,second", [("clip", "clip again"), ("clip", "norm_backward"), ("clip", "log_probs"), ("norm_backward", "norm_backward wide"), ("norm_backward", "log_probs")])
def test_two_threads(gpu, D, rng, first, second):
    kept, made = calls(D, rng)
    failures = []
    threads = [threading.Thread(target=made[name].repeat, args=(200, failures)) for name in (first, second)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, failures[:5]
    assert kept

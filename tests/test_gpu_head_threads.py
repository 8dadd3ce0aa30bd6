"""GPU: the head's loss and distillation called from two host threads at once (ctypes
releases the interpreter lock), at sizes whose kernels need different amounts of
shared memory, of the same kernel."""
import threading

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def together(*calls, times=150):
    """each call `times` over in a thread of its own; the results that were not the first one's"""
    first, wrong, errors = [c() for c in calls], [], []

    def loop(i):
        try:
            for _ in range(times):
                if any(not np.array_equal(a, b) for a, b in zip(calls[i](), first[i])):
                    wrong.append(i)
        except Exception as e:   # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=loop, args=(i,)) for i in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    return wrong


def head(M, n, D, V, tied=True, grad=False):
    r = np.random.default_rng(n + D)
    T = M.Tensor.from_numpy
    w = (r.standard_normal((V, D)) / np.sqrt(D)).astype(np.float32)
    x, w, t = T(r.standard_normal((n, D)).astype(np.float32)), T(w if tied else np.ascontiguousarray(w.T)), T(
        r.integers(0, V, n).astype(np.int32))
    return lambda: [a.numpy() for a in M.linear_xent(x, w, t, tied=tied, grad=grad) if a is not None]


@pytest.mark.parametrize("tied", [True, False])
def test_few_rows(M, tied):
    assert not together(head(M, 1, 20000, 96, tied), head(M, 1, 768, 96, tied))


def test_training(M):
    assert not together(head(M, 300, 64, 4000, grad=True), head(M, 20, 32, 100, grad=True), times=50)


def test_distillation(M):
    r = np.random.default_rng(5)
    T = M.Tensor.from_numpy

    def distill(K):
        s, i, e = (T(r.standard_normal((4, 3000)).astype(np.float32)), T(r.integers(0, 3000, (4, K)).astype(np.int32)),
                   T(r.standard_normal((4, K)).astype(np.float32)))
        return lambda: [a.numpy() for a in M.distill(s, i, e, 2.0)]
    assert not together(distill(1000), distill(800))

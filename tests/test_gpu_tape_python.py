"""GPU: the Python results of the affine norm, the head's loss and distillation handed
to the tape (record_layernorm_affine, record_loss): the Tensors stay their owner's,
before and after the backward pass and with a paused tape, and every reference is
released once."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def counts(rt):
    v = [C.c_int64() for _ in range(3)]
    rt.malus_rc_counts(*(C.byref(a) for a in v))
    return [a.value for a in v]


def last_part(M, seed):
    r = np.random.default_rng(seed)
    T = M.Tensor.from_numpy
    f = lambda *s: T(r.standard_normal(s).astype(np.float32))  # noqa: E731
    x, g, b, w = f(20, 24), f(24), f(24), f(50, 24)
    t = T(r.integers(0, 50, 20).astype(np.int32))
    y, st = M.layernorm_affine(x, g, b)
    loss, nll, dy, dw = M.linear_xent(y, w, t)
    return (x, g, b, w, t), (y, st), (loss, nll, dy, dw)


@pytest.mark.parametrize("paused", [False, True])
def test_results_recorded_stay_their_owners(M, rt, paused):
    rt.malus_tape_reset()
    rt.malus_rc_reset()
    (x, g, b, w, t), (y, st), (loss, nll, dy, dw) = last_part(M, 1)
    for p in (x, g, b, w):
        rt.tape_register_leaf(p.h)
    want = M.layernorm_affine_bwd(x, g, st, dy)
    if paused:
        rt.tape_pause()
    M.record_layernorm_affine(x, g, b, y, st)
    M.record_loss((y, w), (dy, dw), loss)
    before = [a.numpy() for a in (st, dy, dw)]
    if paused:
        rt.tape_resume()
    else:
        rt.backward(loss.h)
        got = [M.Tensor(rt.tape_get_grad(p.h)) for p in (x, g, b, w)]
        for a, f in zip(got, (*want, dw)):
            assert np.array_equal(a.numpy(), f.numpy())
        for a in got:
            a.close()
    for a, f in zip((st, dy, dw), before):   # still there, and the same
        assert np.array_equal(a.numpy(), f)
    for a in (x, g, b, w, t, y, st, loss, nll, dy, dw, *want):
        a.close()
    rt.malus_tape_reset()
    retains, releases, allocs = counts(rt)
    assert allocs + retains == releases


def test_distillation_recorded(M, rt):
    r = np.random.default_rng(2)
    T = M.Tensor.from_numpy
    rt.malus_tape_reset()
    lg, ids = T(r.standard_normal((6, 40)).astype(np.float32)), T(r.integers(0, 40, (6, 3)).astype(np.int64))
    te = T(r.standard_normal((6, 3)).astype(np.float32))
    rt.tape_register_leaf(lg.h)
    loss, kl, dl = M.distill(lg, ids, te, 2.0)
    M.record_loss([lg], [dl], loss)
    rt.backward(loss.h)
    assert np.array_equal(M.Tensor(rt.tape_get_grad(lg.h)).numpy(), dl.numpy())
    rt.malus_tape_reset()


def test_a_loss_without_its_gradients_is_refused(M, rt):
    T = M.Tensor.from_numpy
    x, w, t = T(np.ones((3, 4), np.float32)), T(np.ones((5, 4), np.float32)), T(np.zeros(3, np.int32))
    loss, nll, dx, dw = M.linear_xent(x, w, t, grad=False)
    with pytest.raises(ValueError):
        M.record_loss((x, w), (dx, dw), loss)
    with pytest.raises(ValueError):
        M.record_loss((x, w), (loss,), loss)

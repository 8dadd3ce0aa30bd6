"""GPU: the softmax rows of the losses where a row's memory is used twice: gradients
written over the logits they come from, and shared memory that is filled by bulk
copies and, at a row's ends, by element."""
import numpy as np
import pytest

from test_gpu_distill import inputs, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,V", [(16384, 65), (16384, 128), (4000, 250), (3000, 500), (2000, 1000)])
def test_values_do_not_depend_on_the_gradient(M, rt, n, V):
    """a row's nll reads the target's logit, which its gradient overwrites"""
    r = np.random.default_rng(V)
    T = M.Tensor.from_numpy
    x, w = T(r.standard_normal((n, 8)).astype(np.float32)), T(r.standard_normal((V, 8)).astype(np.float32))
    t = T(r.integers(0, V, n).astype(np.int32))
    before = rt.malus_linear_xent_mode(1)
    try:
        alone = M.linear_xent(x, w, t, grad=False)
        for _ in range(20):
            both = M.linear_xent(x, w, t)
            assert np.array_equal(both[1].numpy(), alone[1].numpy()) and np.array_equal(both[0].numpy(), alone[0].numpy())
    finally:
        rt.malus_linear_xent_mode(before)


@pytest.mark.parametrize("V", [2049, 5003, 10006, 20011])
def test_many_rows_of_changing_alignment(M, V):
    """each row starts one to three elements further from a 16-byte boundary than the last,
    so the ring's slots take a row's ends where the row before had its middle"""
    s, ids, te = inputs(1500, V, 5, V, pad=0.2)
    T = M.Tensor.from_numpy
    ts, ti, tt = T(s), T(ids), T(te)
    first = [a.numpy() for a in M.distill(ts, ti, tt, 1.5)]
    rows = np.r_[0:40, 700:740, 1460:1500]
    (_, kl, dl), (_, tk, td) = reference(s[rows], ids[rows], te[rows], 1.5)
    there = (ids >= 0).any(1)
    part = there[rows].sum() / there.sum()   # the gradient's mean is over all counted rows
    assert (np.abs(first[1][rows] - kl) <= tk + 1e-36).all()
    assert (np.abs(first[2][rows] / part - dl) <= td * 1.001 + 1e-36).all()
    for _ in range(10):
        assert all(np.array_equal(a.numpy(), f) for a, f in zip(M.distill(ts, ti, tt, 1.5), first))

"""GPU: the softmax rows of the losses where a row's memory is used twice: gradients
written over the logits they come from."""
import numpy as np
import pytest

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

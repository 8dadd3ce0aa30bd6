"""GPU: the head on rows longer than 1024 (their planes are made in separate passes) and
past the few-row kernels' shared memory, formula and tolerances as in
test_gpu_linear_xent; and the error in the norm at shapes whose three products take each
form: one tile, K slices, rows off 16 bytes."""
import numpy as np
import pytest

from test_gpu_linear_xent import U, both_products, check, inputs, mode, reference, run  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tied", [True, False])
@pytest.mark.parametrize("n,D,V", [(40, 1280, 500), (300, 1600, 1000), (9, 2050, 701), (5, 1281, 3000), (130, 4099, 257),
                                   (8, 3000, 600), (3, 24000, 90)])
@both_products
def test_wide_rows(M, rt, mode, n, D, V, tied):  # noqa: F811
    x, w, t = inputs(n, D, V, n + D + V, np.int64 if V % 2 else np.int32, 0.25 if n > 4 else 0.0)
    ref, tol = reference(x, w, t)
    check(run(M, x, w, t, tied), ref, tol, f"{n}x{D}x{V}")
    loss, nll, _, _ = M.linear_xent(*(M.Tensor.from_numpy(a) for a in (x, w, t)), grad=False)
    check((loss.numpy(), nll.numpy()), ref, tol, "loss alone")
    assert rt.malus_device_error() == 0


@pytest.mark.parametrize("tied", [True, False])
@pytest.mark.parametrize("n,D,V", [(250, 250, 250), (700, 1280, 999), (3000, 96, 1111), (513, 33, 5001)])
@pytest.mark.parametrize("mode", [0], indirect=True)
def test_error_in_the_norm(M, mode, n, D, V, tied):  # noqa: F811
    """within 16 roundings of a half unit, as test_error_is_that_of_f32"""
    x, w, t = inputs(n, D, V, 3 * n)
    ref, _ = reference(x, w, t)
    for g, r in zip(run(M, x, w, t, tied)[1:], ref[1:]):
        assert np.linalg.norm(g - r) <= 16 * U * np.linalg.norm(r)

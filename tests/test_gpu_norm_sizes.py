"""GPU: the affine layer norm at the first and the last length of every way that a row is
held (threads per row x 16-byte groups per thread), forward and backward, by 16-byte
groups and by single elements."""
import pytest

from test_gpu_norm_affine import inputs, reference, run, within

pytestmark = pytest.mark.gpu

STEPS = ((32, 128), (32, 256), (64, 512), (128, 1024), (256, 1536), (512, 2560), (1024, 8192))   # of a class, its last length
EDGES = sorted({e + o for step, top in STEPS for e in range(step, top + 1, step) for o in (-3, -1, 0, 1, 4)
                if e != 3 * 1024 and 1 <= e + o <= 8196} | {3069, 3071, 3073, 3076})   # 128 threads' last, 256 threads' first


@pytest.mark.parametrize("part", range(4))
def test_every_length_class(M, part):
    for D in EDGES[part::4]:
        x, w, b, dy = inputs((19, D), D)
        ref, tol = reference(x, w, b, dy, 1e-5)
        for got, r, t, what in zip(run(M, x, w, b, dy), ref, tol, ("y", "dx", "dweight", "dbias")):
            within(got, r, t, f"{what} {D}")

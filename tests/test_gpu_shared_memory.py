"""GPU: memory shared with another library (Tensor.wrap, __cuda_array_interface__) may
be rewritten by it between two calls: the second one sees the new values, and results
of the first keep the old ones."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture
def torch():
    torch = pytest.importorskip("torch")
    return torch


def data(shape, seed):
    return np.random.default_rng(seed).standard_normal(shape).astype(np.float32)


def matmul(M, rt, a, b):
    return M.Tensor(rt.tensor_matmul(a.h, b.h)).numpy()


@pytest.mark.parametrize("wrapped", [True, False])
@pytest.mark.parametrize("transposed", [True, False])
def test_a_matmul_after_a_rewrite(M, rt, torch, wrapped, transposed):
    a, b = data((256, 256), 1), M.Tensor.from_numpy(data((256, 256), 2))
    if wrapped:
        there = torch.from_numpy(a).cuda()
        t = M.Tensor.wrap(there.data_ptr(), a.shape)
    else:
        t = M.Tensor.from_numpy(a)
    v = M.Tensor(rt.tensor_permute(t.h, None, 0)) if transposed else t
    torch.cuda.synchronize()
    first = matmul(M, rt, v, b)
    assert np.array_equal(first, matmul(M, rt, M.Tensor.from_numpy(a.T.copy() if transposed else a), b))
    if not wrapped:   # planes were kept before another library saw the memory, too
        there = torch.as_tensor(t, device="cuda")
    there.mul_(-2.0)
    torch.cuda.synchronize()
    assert np.array_equal(matmul(M, rt, v, b), -2.0 * first)
    there.mul_(0.5)
    torch.cuda.synchronize()
    assert np.array_equal(matmul(M, rt, v, b), -first)


def test_products_of_wrapped_memory_are_not_put_off(M, rt, torch):
    a, s, w, m = data((512, 256), 3), data((1,), 4), data((256,), 5), data((512, 256), 6)
    mul, add = getattr(rt, "__broadcast_mul_fwd"), getattr(rt, "__broadcast_add_fwd")
    T = M.Tensor.from_numpy
    there = [torch.from_numpy(v).cuda() for v in (a, s, w, m)]
    torch.cuda.synchronize()
    ta, ts, tw, tm = (M.Tensor.wrap(v.data_ptr(), tuple(v.shape)) for v in there)
    oa, os_, ow = T(a), T(s), T(w)
    got = [M.Tensor(h) for h in (mul(ta.h, ts.h), mul(ta.h, os_.h), mul(oa.h, ts.h), mul(ta.h, tw.h), mul(ta.h, ow.h),
                                 mul(oa.h, tw.h))]
    put_off = M.Tensor(mul(oa.h, os_.h))          # of the runtime's own memory: may be deferred
    got.append(M.Tensor(add(put_off.h, tm.h)))
    for t in (ta, ts, tw, tm):
        t.close()
    rt.gpu_barrier()
    for v in there:
        v.fill_(7.0)                              # the memory is another's again
    torch.cuda.synchronize()
    for g, want in zip(got, (a * s, a * s, a * s, a * w, a * w, a * w, a * s + m)):
        assert np.array_equal(g.numpy(), want)


def test_operators_after_a_rewrite(M, rt, torch):
    x, w = data((300, 64), 7), data((500, 64), 8)
    t = M.Tensor.from_numpy(np.arange(300, dtype=np.int32))
    there = torch.from_numpy(x).cuda()
    torch.cuda.synchronize()
    tx, tw = M.Tensor.wrap(there.data_ptr(), x.shape), M.Tensor.from_numpy(w)
    M.linear_xent(tx, tw, t)
    there.mul_(0.5)
    torch.cuda.synchronize()
    for a, b in zip(M.linear_xent(tx, tw, t), M.linear_xent(M.Tensor.from_numpy(0.5 * x), tw, t)):
        assert np.array_equal(a.numpy(), b.numpy())

"""GPU: the affine layer norm (malus_layernorm_affine_*) against its formula in
64 bits, over every way a row is held (warp, block, re-read), aligned and not,
with and without weight and bias, and through the tape.

Tolerances count roundings of half a unit (u = 2^-24).  A row or column sum
adds at most 48 terms one after another in any thread or level here, so it is
within 48 u of the sum of magnitudes; each formula below adds a few roundings
of its own, rounded up to 64 and 128."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def reference(x, w, b, dy, eps):
    x, dy = x.astype(np.float64), dy.astype(np.float64)
    D = x.shape[-1]
    w = np.ones(D) if w is None else w.astype(np.float64)
    b = np.zeros(D) if b is None else b.astype(np.float64)
    mean = x.mean(-1, keepdims=True)
    rstd = 1.0 / np.sqrt(((x - mean) ** 2).mean(-1, keepdims=True) + eps)
    xh = (x - mean) * rstd
    y = xh * w + b
    g = dy * w
    mg, mgx = g.mean(-1, keepdims=True), (g * xh).mean(-1, keepdims=True)
    dx = rstd * (g - mg - xh * mgx)
    exh = U * (64 * np.abs(x).mean(-1, keepdims=True) * rstd + 32 * np.abs(xh))   # error of xhat
    ty = np.abs(w) * exh + U * (2 * np.abs(xh * w) + 2 * np.abs(y))
    ag = np.abs(g).mean(-1, keepdims=True)
    agx = np.abs(g * xh).mean(-1, keepdims=True)
    tx = rstd * (U * (64 * ag + 8 * np.abs(g) + 128 * np.abs(xh) * agx + 8 * (np.abs(mg) + np.abs(xh * mgx)))
                 + exh * np.abs(mgx) + np.abs(xh) * (np.abs(g) * exh).mean(-1, keepdims=True))
    rows = x.reshape(-1, D).shape[0]
    n = 128 + rows / 100    # additions one after another in a column sum
    f = (-1, D)
    tw = (n * U * np.abs(dy * xh) + np.abs(dy) * exh).reshape(f).sum(0)
    tb = (n * U * np.abs(dy)).reshape(f).sum(0)
    return (y, dx, (dy * xh).reshape(f).sum(0), dy.reshape(f).sum(0)), (ty, tx, tw, tb)


def within(got, ref, tol, what):
    bad = np.abs(got.astype(np.float64) - ref) > tol + 1e-37
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, worst {np.max(np.abs(got - ref) / (tol + 1e-37)):.3g}"


def inputs(shape, seed):
    r = np.random.default_rng(seed)
    D = shape[-1]
    x = (r.standard_normal(shape) * (0.3 + 3 * r.random(shape[:-1] + (1,))) + r.standard_normal(D) * 0.5)
    return (x.astype(np.float32), (1 + 0.3 * r.standard_normal(D)).astype(np.float32),
            r.standard_normal(D).astype(np.float32), r.standard_normal(shape).astype(np.float32))


def run(M, x, w, b, dy, eps=1e-5):
    T = M.Tensor.from_numpy
    tx, td = T(x), T(dy)
    tw = None if w is None else T(w)
    tbi = None if b is None else T(b)
    y, st = M.layernorm_affine(tx, tw, tbi, eps)
    assert st.shape == (x.size // x.shape[-1], 2) and y.shape == x.shape
    return [t.numpy() for t in (y, *M.layernorm_affine_bwd(tx, tw, st, td))]


@pytest.mark.parametrize("shape", [(1, 1), (1, 768), (3, 2), (5, 31), (7, 33), (64, 65), (2, 9, 384), (333, 768),
                                   (1000, 129), (4, 1023), (9, 1024), (9, 1025), (41, 2047), (6, 4096), (5, 5001),
                                   (3, 8191), (3, 8192), (4, 8193), (2, 16384), (3, 16385), (2, 20001), (5000, 17)])
def test_against_the_formula(M, shape):
    x, w, b, dy = inputs(shape, sum(shape))
    ref, tol = reference(x, w, b, dy, 1e-5)
    for got, r, t, what in zip(run(M, x, w, b, dy), ref, tol, ("y", "dx", "dweight", "dbias")):
        within(got, r, t, f"{what} {shape}")


@pytest.mark.parametrize("wb", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("D", [96, 101, 3001])
def test_without_weight_or_bias(M, wb, D):
    x, w, b, dy = inputs((37, D), D)
    w, b = (w if wb[0] else None), (b if wb[1] else None)
    ref, tol = reference(x, w, b, dy, 1e-3)
    for got, r, t, what in zip(run(M, x, w, b, dy, 1e-3), ref, tol, ("y", "dx", "dweight", "dbias")):
        within(got, r, t, what)


def test_gradient_against_differences(M):
    # central differences of sum(y * dy) in 64 bits of the reference's own
    # formula, at the f32 inputs, for a few elements
    x, w, b, dy = inputs((6, 40), 3)
    got = run(M, x, w, b, dy)

    def f(x_, w_, b_):
        x_ = x_.astype(np.float64)
        m = x_.mean(-1, keepdims=True)
        return ((x_ - m) / np.sqrt(x_.var(-1, keepdims=True) + 1e-5) * w_ + b_).ravel() @ dy.astype(np.float64).ravel()

    h = 1e-5
    for (i, j) in [(0, 0), (3, 17), (5, 39)]:
        e = np.zeros_like(x, dtype=np.float64); e[i, j] = h
        num = (f(x + e, w, b) - f(x - e, w, b)) / (2 * h)
        assert abs(num - got[1][i, j]) <= 1e-5 * (1 + abs(num))
        e = np.zeros(40); e[j] = h
        assert abs((f(x, w + e, b) - f(x, w - e, b)) / (2 * h) - got[2][j]) <= 1e-4
        assert abs((f(x, w, b + e) - f(x, w, b - e)) / (2 * h) - got[3][j]) <= 1e-4


def test_views_and_unaligned_memory(M, rt):
    # x as a permuted view; and wrapped memory one float past a 16-byte boundary
    x, w, b, dy = inputs((24, 40), 5)
    ref, tol = reference(x, w, b, dy, 1e-5)
    T = M.Tensor.from_numpy
    xt = T(np.ascontiguousarray(x.T))
    v = M.Tensor(rt.tensor_permute(xt.h, (C.c_size_t * 2)(1, 0), 2))
    y, st = M.layernorm_affine(v, T(w), T(b))
    within(y.numpy(), ref[0], tol[0], "y of a view")
    pad = lambda a: T(np.concatenate([np.zeros(1, np.float32), a.ravel()]))  # noqa: E731
    keep = [pad(x), pad(w), pad(b), pad(dy)]
    ox, ow, ob, od = [M.Tensor.wrap(rt.malus_tensor_data(k.h) + 4, s.shape) for k, s in zip(keep, (x, w, b, dy))]
    y, st = M.layernorm_affine(ox, ow, ob)
    got = (y, *M.layernorm_affine_bwd(ox, ow, st, od))
    for g, r, t, what in zip(got, ref, tol, ("y", "dx", "dweight", "dbias")):
        within(g.numpy(), r, t, what + " unaligned")


def test_no_rows_and_constant_rows(M):
    T = M.Tensor.from_numpy
    w, b = np.ones(8, np.float32), np.arange(8, dtype=np.float32)
    x = T(np.zeros((0, 8), np.float32))
    y, st = M.layernorm_affine(x, T(w), T(b))
    dx, dw, db = M.layernorm_affine_bwd(x, T(w), st, T(np.zeros((0, 8), np.float32)))
    assert y.shape == (0, 8) and dx.shape == (0, 8) and not dw.numpy().any() and not db.numpy().any()
    # a constant row is all bias, its gradient finite
    y, st = M.layernorm_affine(T(np.full((2, 8), 3.0, np.float32)), T(w), T(b))
    assert np.array_equal(y.numpy(), np.tile(b, (2, 1)))


def test_a_bad_row_stays_its_own(M):
    x, w, b, dy = inputs((9, 300), 9)
    clean = run(M, x, w, b, dy)
    x[4, 7] = np.inf
    x[6, 0] = np.nan
    got = run(M, x, w, b, dy)
    keep = [i for i in range(9) if i not in (4, 6)]
    assert np.array_equal(got[0][keep], clean[0][keep]) and np.array_equal(got[1][keep], clean[1][keep])
    assert np.isnan(got[0][6]).all() and np.isnan(got[0][4, 7])


def test_same_bits_every_run_and_in_a_graph(M, rt):
    x, w, b, dy = inputs((777, 768), 11)
    T = M.Tensor.from_numpy
    tx, tw, tbi, td = T(x), T(w), T(b), T(dy)

    def step():
        y, st = M.layernorm_affine(tx, tw, tbi)
        return (y, *M.layernorm_affine_bwd(tx, tw, st, td))
    first = [t.numpy() for t in step()]
    rt.malus_graph_begin()
    outs = step()
    g = rt.malus_graph_end()
    rt.malus_graph_begin()          # a second graph of the same calls: workspaces of its own
    outs2 = step()
    g2 = rt.malus_graph_end()
    for _ in range(2):
        assert rt.malus_graph_replay(g) == 0 and rt.malus_graph_replay(g2) == 0
    for o in (outs, outs2):
        for a, f in zip(o, first):
            assert np.array_equal(a.numpy(), f)
    x2 = x[::-1].copy()
    rt.malus_tensor_write(tx.h, x2.ctypes.data_as(C.c_void_p), x2.nbytes)
    rt.malus_graph_replay(g)
    replayed = [t.numpy() for t in outs]
    rt.malus_graph_destroy(g)
    rt.malus_graph_destroy(g2)
    for a, f in zip(replayed, [t.numpy() for t in step()]):
        assert np.array_equal(a, f)


def test_through_the_tape(M, rt):
    # y used twice, x not a leaf's only path: x -> norm -> y * y -> sum
    x, w, b, _ = inputs((12, 48), 13)
    T = M.Tensor.from_numpy
    rt.malus_tape_reset()
    tx, tw, tbi = T(x), T(w), T(b)
    for t in (tx, tw, tbi):
        rt.tape_register_leaf(t.h)
    st = (C.c_int64 * 1)()
    y = M.Tensor(rt.malus_layernorm_affine_fwd(tx.h, tw.h, tbi.h, 1e-5, st))
    rt.tape_record_layernorm_affine(tx.h, tw.h, tbi.h, y.h, st[0])
    z = M.Tensor(getattr(rt, "__broadcast_mul_fwd")(y.h, y.h))
    rt.tape_record_binop(3, y.h, y.h, z.h)
    s = M.Tensor(getattr(rt, "__reduce_all_sum_fwd")(z.h))
    rt.tape_record_unary(12, z.h, s.h)
    rt.backward(s.h)
    got = [M.Tensor(rt.tape_get_grad(t.h)).numpy() for t in (tx, tw, tbi)]
    yv = y.numpy()
    ref, tol = reference(x, w, b, 2 * yv, 1e-5)
    for g, r, t, what in zip(got, ref[1:], tol[1:], ("dx", "dweight", "dbias")):
        within(g, r, t, what + " of the tape")
    rt.malus_tape_reset()


@pytest.mark.parametrize("D,offs", [(100, (1, 1, 1)), (1101, (3, 3, 3)), (100, (1, 2, 1)), (66, (2, 2, 0)), (2050, (1, 1, 1))])
def test_rows_off_the_16_byte_grid(M, rt, D, offs):
    # x, dy and weight each so many floats past an aligned address; enough rows that a thread walks several
    x, w, b, dy = inputs((3001, D), D)
    ref, tol = reference(x, w, b, dy, 1e-5)
    T = M.Tensor.from_numpy
    keep = [T(np.concatenate([np.zeros(o, np.float32), a.ravel()])) for o, a in zip(offs, (x, dy, w))]
    ox, od, ow = [M.Tensor.wrap(rt.malus_tensor_data(k.h) + 4 * o, s.shape) for k, o, s in zip(keep, offs, (x, dy, w))]
    tb = T(b)
    y, st = M.layernorm_affine(ox, ow, tb)
    got = (y, *M.layernorm_affine_bwd(ox, ow, st, od))
    for g, r, t, what in zip(got, ref, tol, ("y", "dx", "dweight", "dbias")):
        within(g.numpy(), r, t, f"{what} D {D} offsets {offs}")

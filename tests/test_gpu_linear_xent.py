"""GPU: the head with its cross entropy (malus_linear_xent) against its formula
in 64 bits: tied and untied, sizes around every tile edge, several pieces of
tokens, masked rows, i32 and i64 targets, values of very different scale, the
tape, and captured graphs.

Tolerances.  A product sum_k a_k b_k here keeps 22 bits of each operand: every
term is within 1.5 * 2^-22 of itself (two operand roundings and the dropped
product of the low parts), plus 2^-39 of the row's largest element for elements
far below it.  The tensor core truncates: an addition into its accumulator loses
up to 2^-23 of the partial sum, and aligning the 16 products of an instruction
as much again; a chain holds 48 instructions (256 of K) before it is added, rounding
to nearest (2^-24), to the others.  With A = sum |a_k b_k| that bounds the error
by (3 + 96 + K / 512) 2^-23 A.  Plain f32 multiply-adds (mode 1) round once per term
of a chain, which holds all of K or, from 256 on, an eighth of it and the join of
eight: K 2^-24 A at most.  The softmax itself is within (80 + 4 |z|) 2^-24
relative (as in the distillation tests)."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def prod_tol(absa, absb, K):
    """error bound of A B^T for |A| [m, K], |B| [n, K], whichever products compute it"""
    chain = K if K < 256 else K / 8 + 9
    t = max((99 + K / 512) * 2.0 ** -23, chain * U) * (absa @ absb.T)
    t += 2.0 ** -39 * (absa.max(1, initial=0)[:, None] * absb.sum(1)[None] + absa.sum(1)[:, None] * absb.max(1, initial=0)[None])
    return t


def reference(x, w, tgt):
    """w as [V, D]"""
    x, w = x.astype(np.float64), w.astype(np.float64)
    (n, D), V = x.shape, w.shape[0]
    ok = (tgt >= 0) & (tgt < V)
    cnt = max(1, int(ok.sum()))
    x = np.where(ok[:, None], x, 0.0)
    z = x @ w.T
    ez = prod_tol(np.abs(x), np.abs(w), D)
    m = z.max(1, keepdims=True)
    lse = m + np.log(np.exp(z - m).sum(1, keepdims=True))
    q = np.exp(z - lse)
    at = np.where(ok, tgt, 0).astype(np.int64)[:, None]
    nll = np.where(ok, (lse - np.take_along_axis(z, at, 1))[:, 0], 0.0)
    elq = ez + (q * ez).sum(1, keepdims=True) + U * (80 + 8 * np.abs(z - m))   # error of log q
    tn = np.where(ok, np.take_along_axis(elq, at, 1)[:, 0] + 4 * U * (np.abs(m[:, 0]) + np.abs(nll)), 0.0)
    hot = np.zeros_like(q)
    np.put_along_axis(hot, at, 1.0, 1)
    dl = (q - hot) * ok[:, None]
    edl = (q * np.expm1(np.minimum(elq, 1.0)) + 2 * U * np.abs(dl) + 2.0 ** -39) * ok[:, None]
    dx, dw = dl @ w / cnt, dl.T @ x / cnt
    ax, aw, ad = np.abs(x), np.abs(w), np.abs(dl)
    tx = (edl @ aw + prod_tol(ad, aw.T, V) + 4 * U * np.abs(dx) * cnt) / cnt
    tw = (edl.T @ ax + prod_tol(ad.T, ax.T, n) + 8 * U * (ad.T @ ax)) / cnt
    return (np.array([nll.sum() / cnt]), nll, dx, dw), (np.array([tn.sum() / cnt + 2 * U * nll.sum() / cnt]), tn, tx, tw)


def inputs(n, D, V, seed, idt=np.int32, masked=0.0):
    r = np.random.default_rng(seed)
    x = (r.standard_normal((n, D)) * (0.5 + r.random((n, 1)))).astype(np.float32)
    w = (r.standard_normal((V, D)) * 1.5 / np.sqrt(D)).astype(np.float32)
    t = r.integers(0, V, n).astype(idt)
    t[r.random(n) < masked] = -1
    return x, w, t


def run(M, x, w, t, tied=True):
    T = M.Tensor.from_numpy
    wt = T(w if tied else np.ascontiguousarray(w.T))
    loss, nll, dx, dw = [a.numpy() for a in M.linear_xent(T(x), wt, T(t), tied=tied)]
    assert dw.shape == wt.shape and dx.shape == x.shape
    return loss, nll, dx, dw if tied else dw.T


def check(got, ref, tol, msg=""):
    for g, r, t, what in zip(got, ref, tol, ("loss", "nll", "dx", "dweight")):
        bad = ~(np.abs(g - r) <= t + 1e-36)
        assert not bad.any(), f"{what} {msg}: {bad.sum()} of {bad.size} off, worst {np.max(np.abs(g - r) / (t + 1e-36)):.3g}"


SIZES = [(1, 1, 1), (1, 64, 50), (1, 700, 9001), (4, 129, 300), (8, 384, 1000), (3, 5, 2), (7, 33, 65), (64, 64, 64), (65, 63, 129), (128, 128, 256), (129, 130, 257),
         (256, 256, 256), (257, 65, 511), (300, 500, 1007), (511, 257, 300), (1000, 384, 65), (2, 768, 4099),
         (700, 96, 4096), (40, 16, 70001), (9, 24, 131200)]


@pytest.fixture
def mode(request, rt):
    before = rt.malus_linear_xent_mode(request.param)
    yield request.param
    rt.malus_linear_xent_mode(before)


both_products = pytest.mark.parametrize("mode", [-1, 0, 1], indirect=True)


@pytest.mark.parametrize("tied", [True, False])
@pytest.mark.parametrize("n,D,V", SIZES)
@both_products
def test_against_the_formula(M, rt, mode, n, D, V, tied):
    x, w, t = inputs(n, D, V, n + D + V, np.int64 if V % 2 else np.int32, 0.25 if n > 4 else 0.0)
    ref, tol = reference(x, w, t)
    check(run(M, x, w, t, tied), ref, tol, f"{n}x{D}x{V}")
    loss, nll, dx, dw = M.linear_xent(*(M.Tensor.from_numpy(a) for a in (x, w, t)), grad=False)
    check((loss.numpy(), nll.numpy()), ref, tol, "loss alone")
    assert dx is None and dw is None and rt.malus_device_error() == 0


@pytest.mark.parametrize("mode", [0], indirect=True)
def test_error_is_that_of_f32(M, mode):
    """in the norm, the long sums over the vocabulary and over the tokens stay within
    16 roundings of a half unit, far below what the worst case above allows: a chain of
    truncations over K = 20000 would lose over 1e-5 here"""
    x, w, t = inputs(600, 128, 20000, 1)
    ref, _ = reference(x, w, t)
    for g, r in zip(run(M, x, w, t)[1:], ref[1:]):
        assert np.linalg.norm(g - r) <= 16 * U * np.linalg.norm(r)
    x, w, t = inputs(20000, 64, 130, 2)
    ref, _ = reference(x, w, t)
    for g, r in zip(run(M, x, w, t)[1:], ref[1:]):
        assert np.linalg.norm(g - r) <= 16 * U * np.linalg.norm(r)


def test_several_pieces(M, rt):
    # 50304 columns: 2560 rows fill the scratch, so 2700 rows take two pieces
    x, w, t = inputs(2700, 32, 50304, 3, masked=0.5)
    T = M.Tensor.from_numpy
    loss, nll, dx, dw = [a.numpy() for a in M.linear_xent(T(x), T(w), T(t))]
    ref, tol = reference(x[2500:], w, t[2500:])   # a slice of the rows, past the seam
    ok = max(1, (t >= 0).sum())
    part = max(1, (t[2500:] >= 0).sum())
    assert (np.abs(nll[2500:] - ref[1]) <= tol[1] + 1e-36).all()
    assert (np.abs(dx[2500:] * (ok / part) - ref[2]) <= tol[2] * 1.001 + 1e-36).all()
    # dweight is the sum of the pieces' own
    a = [v.numpy() for v in M.linear_xent(T(x[:1500]), T(w), T(t[:1500]))]
    b = [v.numpy() for v in M.linear_xent(T(x[1500:]), T(w), T(t[1500:]))]
    na, nb = (t[:1500] >= 0).sum(), (t[1500:] >= 0).sum()
    both = (a[3].astype(np.float64) * na + b[3].astype(np.float64) * nb) / ok
    assert np.linalg.norm(dw - both) <= 48 * U * np.linalg.norm(both)   # three results within 16 each
    assert rt.malus_device_error() == 0


@both_products
def test_values_of_very_different_scale(M, mode):
    # rows of x over 60 binades and a weight row and column far from the rest:
    # each result row keeps the accuracy of its own magnitudes
    x, w, t = inputs(200, 70, 300, 4)
    x *= np.exp2(np.linspace(-40, 3, 200)).astype(np.float32)[:, None]
    w[17] *= 2.0 ** -30
    w[:, 3] *= 2.0 ** -30
    ref, tol = reference(x, w, t)
    for tied in (True, False):
        check(run(M, x, w, t, tied), ref, tol, "scales")
    # magnitudes whose row scales alone leave the floats' range
    big, small = (x * np.float32(2.0 ** 100)), (w * np.float32(2.0 ** -100))
    check(run(M, big, small, t), *reference(big, small, t), "far scales")
    z = np.zeros_like(x)
    loss, nll, dx, dw = run(M, z, w, t)
    assert np.allclose(nll, np.log(300), rtol=1e-6) and not dw.any()


@both_products
def test_masked_rows_may_hold_anything(M, mode):
    x, w, t = inputs(150, 40, 90, 5, np.int64, 0.4)
    clean = run(M, x, w, t)
    bad = x.copy()
    bad[t < 0] = np.nan
    bad[np.flatnonzero(t < 0)[::2]] = np.inf
    for a, b in zip(run(M, bad, w, t), clean):
        assert np.array_equal(a, b)
    assert not clean[2][t < 0].any() and not clean[1][t < 0].any()


@both_products
def test_no_counted_row_and_no_row(M, mode):
    x, w, t = inputs(70, 40, 90, 6)
    for got in (run(M, x, w, np.full_like(t, -1)), run(M, x[:0], w, t[:0]), run(M, x[:0], w, t[:0], False)):
        assert got[0][0] == 0 and not any(a.any() for a in got)


@both_products
def test_targets_out_of_range_are_reported(M, rt, mode):
    x, w, t = inputs(70, 40, 90, 7)
    t[5] = 90
    rt.malus_device_error()
    got = run(M, x, w, t)
    assert rt.malus_device_error() == 4 and rt.malus_device_error() == 0
    check(got, *reference(x, w, t))


@both_products
def test_a_bad_row_stays_its_own(M, mode):
    x, w, t = inputs(300, 70, 300, 8)
    clean = run(M, x, w, t)
    x[100, 3] = np.inf
    got = run(M, x, w, t)
    keep = np.arange(300) != 100
    assert np.array_equal(got[1][keep], clean[1][keep]) and np.array_equal(got[2][keep], clean[2][keep])
    assert np.isnan(got[1][100])


@both_products
def test_gradients_that_are_not_wanted(M, rt, mode):
    x, w, t = inputs(300, 70, 300, 9)
    full = run(M, x, w, t)
    T = M.Tensor.from_numpy
    tx, tw, tt = T(x), T(w), T(t)
    d = (C.c_int64 * 1)()
    loss = M.Tensor(rt.malus_linear_xent(tx.h, tw.h, tt.h, 1, None, d, None))
    assert np.array_equal(M.Tensor(d[0]).numpy(), full[2]) and np.array_equal(loss.numpy(), full[0])
    loss = M.Tensor(rt.malus_linear_xent(tx.h, tw.h, tt.h, 1, None, None, d))
    assert np.array_equal(M.Tensor(d[0]).numpy(), full[3])


@both_products
def test_views_ranks_and_unaligned_memory(M, rt, mode):
    x, w, t = inputs(60, 41, 77, 10)
    ref, tol = reference(x, w, t)
    T = M.Tensor.from_numpy
    pad = lambda a: T(np.concatenate([np.zeros(1, np.float32), a.ravel()]))  # noqa: E731
    kx, kw = pad(x), pad(w)
    ox = M.Tensor.wrap(rt.malus_tensor_data(kx.h) + 4, (3, 20, 41))
    ow = M.Tensor.wrap(rt.malus_tensor_data(kw.h) + 4, w.shape)
    got = [a.numpy() for a in M.linear_xent(ox, ow, T(t.reshape(3, 20)))]
    assert got[2].shape == (3, 20, 41)
    got[2] = got[2].reshape(60, 41)
    check(got, ref, tol, "unaligned")
    wt = T(np.ascontiguousarray(w.T))
    v = M.Tensor(rt.tensor_permute(wt.h, (C.c_size_t * 2)(1, 0), 2))
    check([a.numpy() for a in M.linear_xent(T(x), v, T(t))], ref, tol, "view")


@both_products
def test_gradient_against_differences(M, mode):
    x, w, t = inputs(6, 20, 30, 11, masked=0.3)
    _, _, dx, dw = run(M, x, w, t)
    h = 1e-4
    f = lambda a, b: reference(a, b, t)[0][0][0]  # noqa: E731
    for n, d in [(0, 0), (3, 11), (5, 19)]:
        e = np.zeros((6, 20)); e[n, d] = h
        assert abs((f(x + e, w) - f(x - e, w)) / (2 * h) - dx[n, d]) <= 1e-6
    for v, d in [(0, 0), (int(t.max()), 7), (29, 19)]:
        e = np.zeros((30, 20)); e[v, d] = h
        assert abs((f(x, w + e) - f(x, w - e)) / (2 * h) - dw[v, d]) <= 1e-6


@both_products
def test_same_bits_in_two_graphs(M, rt, mode):
    x, w, t = inputs(700, 96, 1111, 12, masked=0.2)
    T = M.Tensor.from_numpy
    tx, tw, tt = T(x), T(w), T(t)
    first = [a.numpy() for a in M.linear_xent(tx, tw, tt)]
    ev = M.linear_xent(tx, tw, tt, grad=False)[1].numpy()
    graphs = []
    for _ in range(2):
        rt.malus_graph_begin()
        outs = M.linear_xent(tx, tw, tt)
        outs2 = M.linear_xent(tx, tw, tt, grad=False)
        graphs.append((rt.malus_graph_end(), outs, outs2))
    for g, _, _ in graphs * 2:
        assert rt.malus_graph_replay(g) == 0
    for g, outs, outs2 in graphs:
        for a, f in zip(outs, first):
            assert np.array_equal(a.numpy(), f)
        assert np.array_equal(outs2[1].numpy(), ev)
    x2 = np.ascontiguousarray(x[::-1])
    rt.malus_tensor_write(tx.h, x2.ctypes.data_as(C.c_void_p), x2.nbytes)
    rt.malus_graph_replay(graphs[0][0])
    again = [a.numpy() for a in graphs[0][1]]
    for a, f in zip(again, [a.numpy() for a in M.linear_xent(tx, tw, tt)]):
        assert np.array_equal(a, f)
    for g, _, _ in graphs:
        rt.malus_graph_destroy(g)


def test_norm_head_and_distillation_through_the_tape(M, rt):
    """The model's last part as it is trained: affine norm -> tied head with its
    cross entropy, plus 0.5 * distillation of the same logits, gradients of every
    parameter against the chain in 64 bits."""
    r = np.random.default_rng(13)
    n, D, V, K = 150, 48, 333, 8
    x = r.standard_normal((n, D)).astype(np.float32)
    g = (1 + 0.2 * r.standard_normal(D)).astype(np.float32)
    b = (0.1 * r.standard_normal(D)).astype(np.float32)
    w = (r.standard_normal((V, D)) * 1.5 / np.sqrt(D)).astype(np.float32)
    t = r.integers(0, V, n).astype(np.int32)
    t[::7] = -1
    ids = r.integers(0, V, (n, K)).astype(np.int32)
    te = (r.standard_normal((n, K)) * 2).astype(np.float32)
    T = M.Tensor.from_numpy
    rt.malus_tape_reset()
    tx, tg, tb, tw, tt, ti, tte, half = T(x), T(g), T(b), T(w), T(t), T(ids), T(te), T(np.array([0.5], np.float32))
    for p in (tx, tg, tb, tw):
        rt.tape_register_leaf(p.h)
    o1, o2, o3 = ((C.c_int64 * 1)() for _ in range(3))
    y = M.Tensor(rt.malus_layernorm_affine_fwd(tx.h, tg.h, tb.h, 1e-5, o1))
    rt.tape_record_layernorm_affine(tx.h, tg.h, tb.h, y.h, o1[0])
    ce = M.Tensor(rt.malus_linear_xent(y.h, tw.h, tt.h, 1, None, o2, o3))
    rt.tape_record_loss((C.c_int64 * 2)(y.h, tw.h), (C.c_int64 * 2)(o2[0], o3[0]), 2, ce.h)
    wt = M.Tensor(rt.tensor_permute(tw.h, None, 0))
    rt.tape_record_perm(13, tw.h, wt.h, None, 0)
    lg = M.Tensor(rt.tensor_matmul(y.h, wt.h))
    rt.tape_record_binop(0, y.h, wt.h, lg.h)
    kd = M.Tensor(rt.malus_distill(lg.h, ti.h, tte.h, 2.0, None, o1))
    rt.tape_record_loss((C.c_int64 * 1)(lg.h), o1, 1, kd.h)
    hk = M.Tensor(getattr(rt, "__broadcast_mul_fwd")(kd.h, half.h))
    rt.tape_record_binop(3, kd.h, half.h, hk.h)
    loss = M.Tensor(getattr(rt, "__broadcast_add_fwd")(ce.h, hk.h))
    rt.tape_record_binop(1, ce.h, hk.h, loss.h)
    rt.backward(loss.h)
    got = [M.Tensor(rt.tape_get_grad(p.h)).numpy() for p in (tx, tg, tb, tw)]
    # the chain in 64 bits
    X, G, B, W = (a.astype(np.float64) for a in (x, g, b, w))
    mu = X.mean(1, keepdims=True)
    rs = 1 / np.sqrt(X.var(1, keepdims=True) + 1e-5)
    xh = (X - mu) * rs
    Y = xh * G + B
    z = Y @ W.T
    sm = lambda a: np.exp(a - a.max(1, keepdims=True)) / np.exp(a - a.max(1, keepdims=True)).sum(1, keepdims=True)  # noqa: E731
    ok = t >= 0
    dl = sm(z)
    dl[np.arange(n), np.where(ok, t, 0)] -= 1
    dl = dl * ok[:, None] / ok.sum()
    q, p = sm(z / 2), sm(te.astype(np.float64) / 2)
    for k in range(K):
        np.subtract.at(q, (np.arange(n), ids[:, k]), p[:, k])
    dl = dl + 0.5 * 2.0 * q / n
    dy, dw = dl @ W, dl.T @ Y
    gg = dy * G
    dx = rs * (gg - gg.mean(1, keepdims=True) - xh * (gg * xh).mean(1, keepdims=True))
    want = (dx, (dy * xh).sum(0), dy.sum(0), dw)
    val = np.log(np.exp(z - z.max(1, keepdims=True)).sum(1)) + z.max(1) - z[np.arange(n), np.where(ok, t, 0)]
    lq = np.log(sm(z / 2))[np.arange(n)[:, None], ids]
    kl = 4 * (p * (np.log(p) - lq)).sum(1).mean()
    assert abs(loss.numpy()[0] - ((val * ok).sum() / ok.sum() + 0.5 * kl)) <= 1e-5
    # every link is within the tolerances tested above; in the norm they come to a
    # few hundred half units (the 3xTF32 matmul of the distillation branch: 52 * 2)
    for a, r_, what in zip(got, want, ("x", "weight", "bias", "head")):
        assert np.linalg.norm(a - r_) <= 512 * U * np.linalg.norm(r_), what
    rt.malus_tape_reset()


def test_paused_tape_takes_and_drops_the_gradients(M, rt):
    x, w, t = inputs(20, 8, 30, 14)
    T = M.Tensor.from_numpy
    rt.malus_tape_reset()
    tx, tw, tt = T(x), T(w), T(t)
    a, b = (C.c_int64 * 1)(), (C.c_int64 * 1)()
    live = (C.c_int64 * 3)()
    rt.malus_rc_reset()
    rt.tape_pause()
    loss = M.Tensor(rt.malus_linear_xent(tx.h, tw.h, tt.h, 1, None, a, b))
    rt.tape_record_loss((C.c_int64 * 2)(tx.h, tw.h), (C.c_int64 * 2)(a[0], b[0]), 2, loss.h)
    rt.tape_resume()
    loss.close()
    rt.malus_rc_counts(C.cast(live, C.POINTER(C.c_int64)), C.cast(C.byref(live, 8), C.POINTER(C.c_int64)),
                       C.cast(C.byref(live, 16), C.POINTER(C.c_int64)))
    assert live[2] + live[0] == live[1]     # every allocation and retain was released
    rt.malus_tape_reset()

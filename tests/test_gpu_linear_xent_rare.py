"""GPU: the head's weight gradient of vocabulary entries that are hardly ever
predicted, entry by entry.  Their softmax gradients are 1e-5 to 1e-20 in every
token, and an optimiser that divides by a gradient's own size sees each row at
full scale, so every row of dweight is held to its own magnitudes.

Tolerances (u = 2^-24).  x and weight hold small multiples of 1/2: every product
and sum of the logits is exact, so log q carries only the softmax's own error,
(80 + 8 |z - max|) u as in the distillation tests, and dl = q - onehot that error
of q and two roundings.  No absolute error is allowed for: the products' bound
(prod_tol) is relative to the terms and to the largest one of the row."""
import ctypes as C

import numpy as np
import pytest

from test_gpu_linear_xent import U, both_products, mode, prod_tol, run  # noqa: F401

pytestmark = pytest.mark.gpu


def inputs(n, D, V, seed):
    r = np.random.default_rng(seed)
    x = r.choice(np.array([-2, -1, 1, 2], np.float32), (n, D))
    w = r.choice(np.array([-0.5, 0, 0.5], np.float32), (V, D))
    x[:, 0] = 1.0
    w[:, 0] = -np.floor(30.0 * np.arange(V) / V)   # the later an entry, the rarer
    t = r.integers(0, max(1, V // 4), n).astype(np.int32)
    t[r.random(n) < 0.2] = -1
    return x, w, t


def reference(x, w, t):
    x, w = x.astype(np.float64), w.astype(np.float64)
    n = x.shape[0]
    ok = t >= 0
    cnt = max(1, int(ok.sum()))
    z = x @ w.T
    z -= z.max(1, keepdims=True)
    lq = z - np.log(np.exp(z).sum(1, keepdims=True))
    q = np.exp(lq) * ok[:, None]
    dl = q.copy()
    dl[np.arange(n)[ok], t[ok]] -= 1
    edl = q * U * (80 + 8 * np.abs(z)) + 2 * U * np.abs(dl)
    ad, ax = np.abs(dl), np.abs(x)
    tw = (edl.T @ ax + prod_tol(ad.T, ax.T, n) + 8 * U * (ad.T @ ax)) / cnt
    return dl.T @ x / cnt, tw


@pytest.mark.parametrize("tied", [True, False])
@pytest.mark.parametrize("n,D,V", [(700, 32, 4000), (257, 33, 1001), (20000, 32, 300), (300, 16, 70001), (64, 20, 90)])
@both_products
def test_rows_of_rare_entries(M, rt, mode, n, D, V, tied):  # noqa: F811
    x, w, t = inputs(n, D, V, n + V)
    want, tol = reference(x, w, t)
    dw = run(M, x, w, t, tied)[3]
    assert (np.abs(want).max(1) < 2.0 ** -38).any() or V < 1000   # entries below any fixed grid are among them
    bad = ~(np.abs(dw - want) <= tol + 1e-36)
    assert not bad.any(), f"{bad.any(1).sum()} of {V} rows off, worst {np.max(np.abs(dw - want) / (tol + 1e-36)):.3g}"
    assert rt.malus_device_error() == 0


@pytest.mark.parametrize("tied", [True, False])
def test_a_vocabulary_past_the_piece_bound(M, rt, tied):
    """over 2^21 entries a piece is 64 rows whatever its size: two pieces here, the second
    of six rows, formula and tolerances as above, ten rows at a time"""
    n, D, V = 70, 8, (1 << 21) + 1001
    x, w, t = inputs(n, D, V, 1)
    loss, nll, dx, dw = run(M, x, w, t, tied)
    assert rt.malus_device_error() == 0
    X, W = x.astype(np.float64), w.astype(np.float64)
    cnt = int((t >= 0).sum())
    want, tol, largest = np.zeros((V, D)), np.zeros((V, D)), np.zeros(V)
    for r0 in range(0, n, 10):
        s = slice(r0, r0 + 10)
        ok = t[s] >= 0
        z = X[s] @ W.T
        m = z.max(1, keepdims=True)
        z -= m
        lse = np.log(np.exp(z).sum(1, keepdims=True))
        zt = z[np.arange(10), np.where(ok, t[s], 0)]
        assert (np.abs(nll[s] - np.where(ok, lse[:, 0] - zt, 0)) <= U * (100 + 12 * np.abs(zt))).all()
        q = np.exp(z - lse) * ok[:, None]
        edl = q * U * (80 + 8 * np.abs(z))
        q[np.arange(10)[ok], t[s][ok]] -= 1
        edl += 2 * U * np.abs(q)
        ad, ax = np.abs(q), np.abs(X[s])
        want += q.T @ X[s] / cnt
        tol += (edl.T @ ax + (ad.T @ ax) * (99 * 2.0 ** -23 + 8 * U) + 2.0 ** -39 * 2 * ad.sum(0)[:, None]) / cnt
        largest = np.maximum(largest, ad.max(0))
        tx = (edl @ np.abs(W) + (99 + V / 512) * 2.0 ** -23 * (ad @ np.abs(W)) + 2.0 ** -39 *
              (ad.max(1)[:, None] * np.abs(W).sum(0) + ad.sum(1)[:, None] * np.abs(W).max(0))) / cnt
        assert (np.abs(dx[s] - q @ W / cnt) <= tx * 1.001 + 1e-36).all()
    tol += 2.0 ** -39 * largest[:, None] * np.abs(X).sum(0) / cnt
    assert (np.abs(dw - want) <= tol + 1e-36).all()


@pytest.mark.parametrize("tied", [True, False])
def test_one_gradient_alone_over_several_pieces(M, rt, tied):
    """with one gradient the planes lie over the logits, with both only dweight's do: the
    same bits either way, over two pieces"""
    x, w, t = inputs(2700, 16, 50304, 3)
    T = M.Tensor.from_numpy
    tx, tw, tt = T(x), T(w if tied else np.ascontiguousarray(w.T)), T(t)
    loss, nll, dx, dw = M.linear_xent(tx, tw, tt, tied=tied)
    for i, both in ((1, dx), (2, dw)):
        out = [(C.c_int64 * 1)() for _ in range(3)]
        rt.tensor_release(rt.malus_linear_xent(tx.h, tw.h, tt.h, int(tied), out[0], *(out[k] if k == i else None for k in (1, 2))))
        got = [M.Tensor(out[0][0]), M.Tensor(out[i][0])]
        assert np.array_equal(got[0].numpy(), nll.numpy()) and np.array_equal(got[1].numpy(), both.numpy())
    assert rt.malus_device_error() == 0

"""GPU: distillation from a teacher's top logits (malus_distill) against its
formula in 64 bits: rows of a warp, rows that stay in a block's shared memory and
longer ones, aligned and not, ragged, repeated and missing entries, i32 and i64 ids, and the tape.

Tolerances (u = 2^-24): a base-2 exponential argument z = (s - max) * c carries
3 roundings, so exp has a relative error of 3 u |z| + 4 u (exp2f is within two
units); the sum Z adds at most 64 terms one after another in any thread or
level.  So q is within (80 + 4 |z|) u relative, log q within (80 + 8 |z|) u,
and the same holds for p."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def reference(s, ids, te, T):
    s, te = s.astype(np.float64) / T, te.astype(np.float64) / T
    N, V = s.shape
    there = (ids >= 0) & (ids < V) & (te != -np.inf)
    counted = there.any(1)
    cnt = max(1, counted.sum())
    kl, dl = np.zeros(N), np.zeros((N, V))
    tk, td = np.zeros(N), np.zeros((N, V))
    for n in range(N):
        if not counted[n]:
            continue
        i, t = ids[n][there[n]].astype(np.int64), te[n][there[n]]
        z, zt = s[n] - s[n].max(), t - t.max()
        lq = z - np.log(np.exp(z).sum())
        lp = zt - np.log(np.exp(zt).sum())
        q, p = np.exp(lq), np.exp(lp)
        kl[n] = T * T * (p * (lp - lq[i])).sum()
        tk[n] = T * T * U * (p * (160 + 16 * (np.abs(lp) + np.abs(lq[i])))).sum()
        with np.errstate(invalid="ignore"):   # exp(-inf) = 0 carries no error
            td[n] = np.where(q > 0, q * (96 + 8 * np.abs(z)), 0.0)
        np.add.at(td[n], i, p * (96 + 8 * np.abs(zt)) + p)
        td[n] *= U * T / cnt
        dl[n] = q
        np.subtract.at(dl[n], i, p)
        dl[n] *= T / cnt
    return (np.array([kl.sum() / cnt]), kl, dl), (np.array([tk.sum() / cnt + U * abs(kl.sum() / cnt)]), tk, td)


def inputs(N, V, K, seed, idt=np.int32, pad=0.0):
    r = np.random.default_rng(seed)
    s = (r.standard_normal((N, V)) * 2).astype(np.float32)
    ids = r.integers(0, V, (N, K)).astype(idt)
    te = (r.standard_normal((N, K)) * 2 + 5).astype(np.float32)
    ids[r.random((N, K)) < pad] = -1
    return s, ids, te


def run(M, s, ids, te, T):
    t = M.Tensor.from_numpy
    loss, kl, dl = M.distill(t(s), t(ids), t(te), T)
    loss2, kl2, none = M.distill(t(s), t(ids), t(te), T, grad=False)
    out = loss.numpy(), kl.numpy(), dl.numpy()
    assert none is None and np.array_equal(loss2.numpy(), out[0], equal_nan=True)
    assert np.array_equal(kl2.numpy(), out[1], equal_nan=True)
    return out


def check(got, ref, tol, msg=""):
    for g, r, t, what in zip(got, ref, tol, ("loss", "kl", "dlogits")):
        bad = ~(np.abs(g - r) <= t + 1e-36)
        assert not bad.any(), f"{what} {msg}: {bad.sum()} of {bad.size} off, worst {np.max(np.abs(g - r) / (t + 1e-36)):.3g}"


@pytest.mark.parametrize("N,V,K,T,idt,pad", [
    (1, 1, 1, 1.0, np.int32, 0.0), (3, 5, 2, 0.5, np.int64, 0.0), (33, 65, 8, 2.0, np.int32, 0.3),
    (5, 1000, 64, 1.0, np.int32, 0.9), (4, 10007, 20, 3.0, np.int64, 0.2), (3, 16381, 7, 1.5, np.int32, 0.0),
    (3, 16384, 33, 1.0, np.int32, 0.0), (2, 16385, 33, 1.0, np.int32, 0.0), (5, 32003, 20, 1.0, np.int64, 0.3),
    (3, 50304, 64, 2.0, np.int32, 0.0), (2, 65537, 100, 1.0, np.int32, 0.1), (2, 140001, 1024, 2.0, np.int64, 0.1),
    (3, 262143, 3, 1.0, np.int32, 0.0), (2, 57597, 9, 1.0, np.int32, 0.0), (301, 57603, 9, 1.0, np.int32, 0.3), (2000, 33, 4, 2.0, np.int32, 0.5)])
def test_against_the_formula(M, N, V, K, T, idt, pad):
    s, ids, te = inputs(N, V, K, N + V + K, idt, pad)
    check(run(M, s, ids, te, T), *reference(s, ids, te, T), f"N {N} V {V} K {K}")


@pytest.mark.parametrize("V", [100, 20001])
def test_repeated_and_missing_entries(M, V):
    s, ids, te = inputs(6, V, 6, V)
    ids[0] = 7                                   # the same id six times
    ids[1, 3:] = ids[1, :3]                      # three ids twice
    ids[2] = -1                                  # no entry: the row is not counted
    te[3] = -np.inf                              # nor here
    te[4, 2:] = -np.inf
    s[5, 1::2] = -np.inf                         # masked vocabulary, entries on the rest
    ids[5] = ids[5] // 2 * 2
    s[2] = np.nan                                # not looked at
    te[1, 0] = -np.inf
    got = run(M, s, ids, te, 1.0)
    s[2] = 0
    ref, tol = reference(s, ids, te, 1.0)
    check(got, ref, tol)
    assert got[1][2] == 0 and got[1][3] == 0 and not got[2][2:4].any()


def test_no_counted_row_and_no_row(M):
    s, ids, te = inputs(4, 50, 3, 1)
    loss, kl, dl = run(M, s, np.full_like(ids, -1), te, 1.0)
    assert loss[0] == 0 and not kl.any() and not dl.any()
    loss, kl, dl = run(M, s[:0], ids[:0], te[:0], 1.0)
    assert loss[0] == 0 and kl.shape == (0,) and dl.shape == (0, 50)


def test_infinities_give_what_the_formula_gives(M):
    s, ids, te = inputs(4, 20001, 3, 2)
    s[1, 5] = np.nan
    s[2, 9] = np.inf
    s[3, ids[3, 0]] = -np.inf                    # the teacher wants what the student excludes
    loss, kl, dl = run(M, s, ids, te, 1.0)
    assert np.isnan(kl[1]) and np.isnan(dl[1]).all() and np.isnan(kl[2]) and np.isnan(dl[2, 9])
    assert np.isinf(kl[3]) and np.isfinite(dl[3]).all() and np.isfinite(dl[0]).all()


def test_ids_out_of_range_are_reported(M, rt):
    s, ids, te = inputs(3, 40, 4, 3)
    ids[1, 2] = 40
    rt.malus_device_error()
    got = run(M, s, ids, te, 1.0)
    assert rt.malus_device_error() == 4 and rt.malus_device_error() == 0
    check(got, *reference(s, ids, te, 1.0))


def test_views_and_unaligned_memory(M, rt):
    s, ids, te = inputs(7, 1031, 5, 4)
    ref, tol = reference(s, ids, te, 1.0)
    t = M.Tensor.from_numpy
    flat = t(np.concatenate([np.zeros(1, np.float32), s.ravel()]))
    u = M.Tensor.wrap(rt.malus_tensor_data(flat.h) + 4, s.shape)
    check([a.numpy() for a in M.distill(u, t(ids), t(te))], ref, tol, "unaligned")
    st = t(np.ascontiguousarray(s.T))
    v = M.Tensor(rt.tensor_permute(st.h, (C.c_size_t * 2)(1, 0), 2))
    check([a.numpy() for a in M.distill(v, t(ids), t(te))], ref, tol, "view")


def test_gradient_against_differences(M):
    s, ids, te = inputs(5, 40, 4, 6)
    _, _, dl = run(M, s, ids, te, 2.0)
    h = 1e-4
    for n, v in [(0, 0), (2, int(ids[2, 1])), (4, 39)]:
        up, dn = s.astype(np.float64), s.astype(np.float64)
        up[n, v] += h
        dn[n, v] -= h
        num = (reference(up, ids, te, 2.0)[0][0] - reference(dn, ids, te, 2.0)[0][0])[0] / (2 * h)
        assert abs(num - dl[n, v]) <= 1e-6


def test_same_bits_in_two_graphs(M, rt):
    s, ids, te = inputs(65, 20011, 16, 7, pad=0.3)
    t = M.Tensor.from_numpy
    a, b, c = t(s), t(ids), t(te)
    first = [x.numpy() for x in M.distill(a, b, c, 2.0)]
    graphs = []
    for _ in range(2):
        rt.malus_graph_begin()
        outs = M.distill(a, b, c, 2.0)
        graphs.append((rt.malus_graph_end(), outs))
    for g, _ in graphs * 2:
        assert rt.malus_graph_replay(g) == 0
    for g, outs in graphs:
        for x, f in zip(outs, first):
            assert np.array_equal(x.numpy(), f)
        rt.malus_graph_destroy(g)


def test_through_the_tape(M, rt):
    # logits = x @ w, loss = distill(logits) * 3 (so the loss's own gradient is not 1)
    r = np.random.default_rng(8)
    x = r.standard_normal((20, 24)).astype(np.float32)
    w = r.standard_normal((24, 50)).astype(np.float32)
    _, ids, te = inputs(20, 50, 4, 8, pad=0.2)
    t = M.Tensor.from_numpy
    rt.malus_tape_reset()
    tx, tw, ti, tt, three = t(x), t(w), t(ids), t(te), t(np.array([3.0], np.float32))
    rt.tape_register_leaf(tw.h)
    lg = M.Tensor(rt.tensor_matmul(tx.h, tw.h))
    rt.tape_record_binop(0, tx.h, tw.h, lg.h)
    dl = (C.c_int64 * 1)()
    loss = M.Tensor(rt.malus_distill(lg.h, ti.h, tt.h, 2.0, None, dl))
    rt.tape_record_loss((C.c_int64 * 1)(lg.h), dl, 1, loss.h)
    out = M.Tensor(getattr(rt, "__broadcast_mul_fwd")(loss.h, three.h))
    rt.tape_record_binop(3, loss.h, three.h, out.h)
    rt.backward(out.h)
    g = M.Tensor(rt.tape_get_grad(tw.h)).numpy()
    ref = reference(lg.numpy(), ids, te, 2.0)
    want = 3 * x.astype(np.float64).T @ ref[0][2]
    # the products' own rounding (24 and 20 terms) on top of dlogits' tolerance
    tol = 3 * np.abs(x).astype(np.float64).T @ (ref[1][2] + 32 * U * np.abs(ref[0][2]))
    assert (np.abs(g - want) <= tol).all()
    rt.malus_tape_reset()

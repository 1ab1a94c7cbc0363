"""Fused feed-forward products, gradients and clipping on p x q gloo ranks,
against plain formulas in 64 bits (tolerances as in test_ffn.py)."""
import math

import pytest
import torch

import slate_amd as sl
from slate_amd.core.enums import Op
from slate_amd.models.aux import allgather_dense as D

from dist_util import run_dist
from test_ffn import act64, act_bound, u_of, w_of, within


def rnd(m, n, dt, seed, std=1.0):
    return (torch.randn(m, n, generator=torch.Generator().manual_seed(seed), dtype=torch.float64) * std).to(dt)


def spread(X, nb, p, q, trans=False, mb=None):
    """X (logical) as a distributed matrix, stored transposed or not."""
    S = X.t().contiguous() if trans else X
    M = sl.Matrix(S.shape[0], S.shape[1], nb=nb, mb=mb, p=p, q=q, dtype=X.dtype)
    M.insertLocalTiles()
    sl.from_dense(M, S)
    return M.transpose() if trans else M


def _products(rank, size, p, q, dt):
    m, n, k = 37, 29, 43
    u, w = u_of(dt), w_of(dt)
    a, a2, b = rnd(m, k, dt, 1, k ** -.5), rnd(m, k, dt, 2, k ** -.5), rnd(k, n, dt, 3)
    r, g = rnd(m, n, dt, 4), rnd(m, n, dt, 5)
    for (ta, tb, tc, nbA, bias) in [(True, False, False, 8, 1), (False, True, False, 8, 2), (True, False, True, 6, 1),
                                    (False, False, False, 16, 0), (True, True, True, 8, 2)]:
        bv = None if not bias else (rnd(m, 1, dt, 6) if bias == 1 else rnd(1, n, dt, 6))
        A, A2, B = spread(a, nbA, p, q, ta), spread(a2, nbA, p, q, ta), spread(b, 8, p, q, tb)
        Bv = None if bv is None else spread(bv, 8, p, q)
        R, G = spread(r, 8, p, q), spread(g, 8, p, q, tc)
        C, Z = spread(torch.zeros(m, n, dtype=dt), 8, p, q, tc), spread(torch.zeros(m, n, dtype=dt), 8, p, q)
        sl.gemm_bias_act(0.5, A, B, Bv, "gelu", 2.0, R, C, Z)
        z = 0.5 * (a.double() @ b.double()) + (0 if bv is None else bv.double())
        S = 0.5 * (a.double().abs() @ b.double().abs()) + (0 if bv is None else bv.double().abs())
        ez = (k + 4) * w * S
        y = act64("gelu", z)[0] + 2 * r.double()
        ey = 1.13 * ez + act_bound(z, w) + 8 * w * (y.abs() + 2 * r.double().abs())
        within(D(Z), z, ez + u * (z.abs() + ez))
        within(D(C), y, ey + u * (y.abs() + ey))
        # gradients from the stored Z
        dA, dB = spread(torch.zeros(m, k, dtype=dt), nbA, p, q, ta), spread(torch.zeros(k, n, dtype=dt), 8, p, q, tb)
        db = None if bv is None else spread(torch.zeros_like(bv), 8, p, q)
        sl.gemm_bias_act_grad(0.5, A, B, "gelu", Z, G, dA, dB, db)
        zs = D(Z).double()
        dz = g.double() * act64("gelu", zs)[1]
        f = u * dz.abs() + 32 * w * (1 + zs.abs()) * g.double().abs()
        for got, x, y_, fx in ((dA, dz @ b.double().t(), (dz.abs() @ b.double().abs().t()), f @ b.double().abs().t()),
                               (dB, a.double().t() @ dz, a.double().abs().t() @ dz.abs(), a.double().abs().t() @ f)):
            e = 0.5 * (fx + 64 * w * y_)
            within(D(got), 0.5 * x, e + u * (0.5 * x.abs() + e))
        if db is not None:
            d = 1 if bias == 1 else 0
            want = dz.sum(d, keepdim=True)
            e = (32 * w * (1 + zs.abs()) * g.double().abs() + 64 * w * dz.abs()).sum(d, keepdim=True)
            within(D(db), want, e + u * (want.abs() + e))
        # gated
        Z1, Z2 = (spread(torch.zeros(m, n, dtype=dt), 8, p, q) for _ in range(2))
        sl.gemm_gated(A, A2, B, "silu", C, Z1, Z2)
        z1, z2 = a.double() @ b.double(), a2.double() @ b.double()
        e1, e2 = ((k + 4) * w * (x.double().abs() @ b.double().abs()) for x in (a, a2))
        within(D(Z1), z1, e1 + u * (z1.abs() + e1))
        v = act64("silu", z1)[0]
        ev = 1.13 * e1 + act_bound(z1, w)
        ey = ev * z2.abs() + e2 * v.abs() + ev * e2 + 2 * w * (v * z2).abs()
        within(D(C), v * z2, ey + u * ((v * z2).abs() + ey))
        dA2 = spread(torch.zeros(m, k, dtype=dt), nbA, p, q, ta)
        sl.gemm_gated_grad(A, A2, B, "silu", Z1, Z2, G, dA, dA2, dB)
        s1, s2, gd = D(Z1).double(), D(Z2).double(), g.double()
        val, sl_ = act64("silu", s1)
        d1, d2 = gd * s2 * sl_, gd * val
        f1, f2 = u * d1.abs() + 64 * w * (1 + s1.abs()) * (gd * s2).abs(), u * d2.abs() + 64 * w * (1 + s1.abs()) * (gd * s1).abs()
        bt = b.double().t()
        for got, x, f in ((dA, d1, f1), (dA2, d2, f2)):
            want, e = x @ bt, f @ bt.abs() + 64 * w * (x.abs() @ bt.abs())
            within(D(got), want, e + u * (want.abs() + e))
        at, at2 = a.double().t(), a2.double().t()
        want = at @ d1 + at2 @ d2
        e = at.abs() @ f1 + at2.abs() @ f2 + 128 * w * (at.abs() @ d1.abs() + at2.abs() @ d2.abs())
        within(D(dB), want, e + u * (want.abs() + e))
    # a block of a larger matrix, off the tile borders, as output
    big = spread(rnd(m + 11, n + 9, dt, 8), 8, p, q)
    keep = D(big).clone()
    sl.gemm_bias_act(1.0, spread(a, 8, p, q), spread(b, 8, p, q), None, "relu", 0.0, None, big.slice(5, 5 + m - 1, 3, 3 + n - 1))
    out = D(big)
    z = a.double() @ b.double()
    e = (k + 4) * w * (a.double().abs() @ b.double().abs())
    within(out[5:5 + m, 3:3 + n], z.clamp(min=0), e + u * (z.abs() + e))
    out[5:5 + m, 3:3 + n] = keep[5:5 + m, 3:3 + n]
    assert torch.equal(out, keep)
    # alpha = 0, and rectangular tiles
    C = spread(torch.zeros(m, n, dtype=dt), 8, p, q, mb=5)
    sl.gemm_bias_act(0.0, spread(a, 8, p, q), spread(b, 8, p, q), None, "identity", 1.0, spread(r, 8, p, q), C)
    assert torch.equal(D(C), r)


@pytest.mark.parametrize("p,q", [(2, 1), (1, 2), (2, 2)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_products(p, q, dt):
    run_dist(_products, p * q, p, q, dt)


def _clip(rank, size, p, q):
    for dt, out in ((torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.float64, torch.float64),
                    (torch.float16, torch.float16)):
        xs = [rnd(m, n, dt, i) for i, (m, n) in enumerate([(37, 29), (5, 64), (1, 3), (70, 1)])]
        s = math.sqrt(sum(float((x.double() ** 2).sum()) for x in xs))
        A = [spread(x, 8, p, q) for x in xs]
        B = [spread(torch.zeros(x.shape, dtype=out), 8, p, q) for x in xs]
        got = sl.clip_norm(2.0, A, B)
        assert abs(float(got) - s) <= 1e-12 * s
        for x, b in zip(xs, B):
            want = x.double() * (2.0 / s)
            assert ((D(b).double() - want).abs() <= (u_of(out) + 4 * w_of(out) + 1e-12) * want.abs() + 1e-8 * (out == torch.float16)).all()
        if dt == out:
            sl.clip_norm(2.0, A)
            for a, b in zip(A, B):
                assert torch.equal(D(a), D(b))
        assert abs(sl.global_norm(B) - 2.0) <= 1e-2
    with pytest.raises(sl.SlateError):
        sl.clip_norm(1.0, A, [spread(x, 4, p, q) for x in xs])


@pytest.mark.parametrize("p,q", [(2, 1), (2, 2)])
def test_clip(p, q):
    run_dist(_clip, p * q, p, q)


def _refused(call, match="overlap"):
    with pytest.raises(sl.SlateError, match=match):
        call()


def _overlaps(rank, size, p, q):
    """Outputs that share elements with other matrices are refused on every
    rank, as on one; nothing is written."""
    dt, n = torch.float64, 16
    mats = [rnd(n, n, dt, i) for i in range(8)]
    A, A2, B, R, C, Z, G, X = M = [spread(x, 4, p, q) for x in mats]
    none = None
    for call in (lambda: sl.gemm_bias_act_grad(1.0, A, B, "gelu", Z, G, A, X, none),
                 lambda: sl.gemm_bias_act_grad(1.0, A, B, "gelu", Z, G, X, X, none),
                 lambda: sl.gemm_bias_act_grad(1.0, A, B, "gelu", Z, G, X, Z, none),
                 lambda: sl.gemm_bias_act_grad(1.0, A, B, "gelu", Z, G, none, none, G.slice(0, n - 1, 3, 3)),
                 lambda: sl.gemm_bias_act(1.0, A, B, none, "gelu", 0.0, none, C, C),
                 lambda: sl.gemm_bias_act(1.0, A, B, none, "gelu", 0.0, none, A),
                 lambda: sl.gemm_bias_act(1.0, A, B, none, "gelu", 0.0, none, A.transpose()),
                 lambda: sl.gemm_bias_act(1.0, A, B, none, "gelu", 1.0, C.transpose(), C),
                 lambda: sl.gemm_bias_act(1.0, A, B, C.slice(0, n - 1, 2, 2), "gelu", 1.0, none, C),
                 lambda: sl.gemm_bias_act(1.0, A.slice(0, 7, 0, n - 1), B, none, "gelu", 1.0, C.slice(1, 8, 0, n - 1),
                                          C.slice(0, 7, 0, n - 1)),
                 lambda: sl.gemm_gated(A, A2, B, "silu", C, Z, Z), lambda: sl.gemm_gated(A, A2, B, "silu", B),
                 lambda: sl.gemm_gated_grad(A, A2, B, "silu", Z, C, G, A, R, X),
                 lambda: sl.gemm_gated_grad(A, A2, B, "silu", Z, C, G, R, R, X),
                 lambda: sl.clip_norm(1.0, [A, A]), lambda: sl.clip_norm(1.0, [A, B], [X, A]),
                 lambda: sl.clip_norm(1.0, [A.slice(0, 4, 0, 4), A.slice(4, 8, 4, 8)]),
                 lambda: sl.clip_norm(1.0, [A, A.slice(n - 1, n - 1, n - 1, n - 1)])):   # one rank's element
        _refused(call)
    for x, m in zip(mats, M):
        assert torch.equal(D(m), x)
    # blocks of one matrix that lie apart, the residual's own matrix, and scaling into itself are taken
    sl.gemm_bias_act(1.0, A, B, none, "identity", 1.0, R, R)
    within(D(R), mats[3] + mats[0] @ mats[2], 40 * 2.0 ** -53 * (mats[3].abs() + mats[0].abs() @ mats[2].abs()))
    sl.gemm_bias_act(1.0, A.slice(0, 7, 0, 7), A.slice(0, 7, 8, 15), none, "relu", 0.0, none, A.slice(8, 15, 0, 7))
    want = (mats[0][:8, :8] @ mats[0][:8, 8:]).clamp(min=0)
    within(D(A)[8:, :8], want, 40 * 2.0 ** -53 * (mats[0][:8, :8].abs() @ mats[0][:8, 8:].abs()) + 1e-300)
    s = float(sl.clip_norm(1.0, [B, C.slice(0, 7, 0, 15), C.slice(8, 15, 0, 15)],
                           [B, X.slice(0, 7, 0, 15), X.slice(8, 15, 0, 15)]))
    want = math.sqrt(float((mats[2] ** 2).sum() + (mats[4] ** 2).sum()))
    assert abs(s - want) <= 1e-12 * want
    assert float((D(X) - mats[4] / want).abs().max()) <= 1e-15


@pytest.mark.parametrize("p,q", [(2, 1), (2, 2)])
def test_overlaps(p, q):
    run_dist(_overlaps, p * q, p, q)


def _own_buffers(rank, size):
    """Buffers of the caller that overlap on one rank only: every rank is told
    (clipping: that rank, and the others' norm is NaN), none waits for another."""
    n, dt = 16, torch.float64
    buf = torch.randn(n // size * n * 2, generator=torch.Generator().manual_seed(rank), dtype=dt)
    was = buf.clone()
    half = n // size * n

    def wrap(first):
        return sl.Matrix.fromScaLAPACK(n, n, buf[first:first + half].view(n, n // size).t(), nb=4, p=size, q=1)

    A, B = wrap(0), wrap(half if rank == 0 else half - 8)
    E, F = (spread(rnd(n, n, dt, i), 4, size, 1) for i in (1, 2))
    _refused(lambda: sl.gemm_bias_act(1.0, A, E, None, "relu", 0.0, None, B))
    _refused(lambda: sl.gemm_bias_act_grad(1.0, A, E, "relu", F, F, B, None, None))
    _refused(lambda: sl.gemm_gated_grad(A, E, E, "relu", F, F, F, None, None, B))
    if rank == 0:
        assert math.isnan(float(sl.clip_norm(1.0, [A, B])))
    else:
        _refused(lambda: sl.clip_norm(1.0, [A, B]))
    assert torch.equal(buf, was)
    A, B = wrap(0), wrap(half)
    sl.gemm_bias_act(1.0, E, F, None, "identity", 0.0, None, B)
    e, f = rnd(n, n, dt, 1), rnd(n, n, dt, 2)
    within(D(B), e @ f, 40 * 2.0 ** -53 * (e.abs() @ f.abs()))
    assert torch.equal(buf[:half], was[:half])


def test_own_buffers():
    run_dist(_own_buffers, 2)


def _one_of(rank, size):
    """Matrices on one rank of a larger communicator: the others take part without elements."""
    m, n, k, dt = 12, 9, 10, torch.float64
    a, a2, b, r, g = rnd(m, k, dt, 1), rnd(m, k, dt, 2), rnd(k, n, dt, 3), rnd(m, n, dt, 4), rnd(m, n, dt, 5)
    A, A2, B, R, G, C, Z, Z2 = (spread(x, 4, 1, 1) for x in (a, a2, b, r, g, 0 * r, 0 * r, 0 * r))
    tol = 400 * 2.0 ** -53
    for bias in (rnd(m, 1, dt, 6), rnd(1, n, dt, 6), None):
        bv = None if bias is None else spread(bias, 4, 1, 1)
        sl.gemm_bias_act(1.0, A, B, bv, "gelu", 1.0, R, C, Z)
        z = a @ b + (0 if bias is None else bias)
        y, s = act64("gelu", z)
        assert float((D(Z) - z).abs().max()) <= tol * 10 and float((D(C) - y - r).abs().max()) <= tol * 10
        dA, dB, db = spread(0 * a, 4, 1, 1), spread(0 * b, 4, 1, 1), None if bv is None else spread(0 * bias, 4, 1, 1)
        sl.gemm_bias_act_grad(1.0, A, B, "gelu", Z, G, dA, dB, db)
        dz = g * s
        assert float((D(dA) - dz @ b.t()).abs().max()) <= tol * 100 and float((D(dB) - a.t() @ dz).abs().max()) <= tol * 100
        if db is not None:
            d = 1 if bias.shape[1] == 1 else 0
            assert float((D(db) - dz.sum(d, keepdim=True)).abs().max()) <= tol * 100
    sl.gemm_gated(A, A2, B, "silu", C, Z, Z2)
    v, s = act64("silu", a @ b)
    assert float((D(C) - v * (a2 @ b)).abs().max()) <= tol * 100
    sl.gemm_gated_grad(A, A2, B, "silu", Z, Z2, G, None, None, dB)
    want = a.t() @ (g * (a2 @ b) * s) + a2.t() @ (g * v)
    assert float((D(dB) - want).abs().max()) <= tol * 1000
    # refusals are every rank's
    long = spread(rnd(m + 1, 1, dt, 6), 4, 1, 1)
    _refused(lambda: sl.gemm_bias_act(1.0, A, B, long, "gelu", 1.0, R, C, Z), "bias")
    _refused(lambda: sl.gemm_bias_act(1.0, B, A, None, "gelu", 1.0, R, C, Z), "wanted")
    _refused(lambda: sl.gemm_bias_act_grad(1.0, A, B, "gelu", Z, G, dA, dB, long), "bias")
    _refused(lambda: sl.gemm_gated(A, A2, B, "silu", C, Z, Z))
    _refused(lambda: sl.gemm_gated_grad(A, A2, B, "silu", Z, Z2, G, A, None, dB))
    # no rank waits for another: the one with the elements may call alone
    if rank == 0:
        sl.gemm_bias_act(1.0, A, B, bv, "gelu", 1.0, R, C, Z)
    # another communicator
    from slate_amd.parallel.comm import self_comm
    own = sl.Matrix.fromLAPACK(m, n, torch.zeros(n, m, dtype=dt).t(), nb=4, comm=self_comm())
    _refused(lambda: sl.gemm_bias_act(1.0, A, B, None, "gelu", 0.0, None, own), "communicator")
    two = spread(0 * r, 4, size, 1)
    _refused(lambda: sl.gemm_bias_act(1.0, A, B, None, "gelu", 1.0, own, two), "communicator")
    sl.gemm_bias_act(1.0, A, B, None, "identity", 0.0, None, two)
    assert float((D(two) - a @ b).abs().max()) <= tol * 10


def test_one_of_two():
    run_dist(_one_of, 2)


def _precise(rank, size, p, q, dt):
    m, n, k = 37, 29, 43
    u, w = u_of(dt), w_of(dt)
    a, a2, b, z1, z2, g = (rnd(*s, dt, i) for i, s in enumerate(((m, k), (m, k), (k, n), (m, n), (m, n), (m, n))))
    A, A2, B, Z1, Z2, G = (spread(x, 8, p, q) for x in (a, a2, b, z1, z2, g))
    dA, dA2, dB, db = (spread(0 * x, 8, p, q) for x in (a, a, b, a[:, :1]))
    opts = {"PreciseGradient": True}
    a, a2, b, z1, z2, g = (x.double() for x in (a, a2, b, z1, z2, g))
    for gated in (False, True):
        v, s = act64("silu", z1)
        c = g * z2 if gated else g
        dz = [c * s] + [g * v] * gated
        f = [(u * u + 4 * w) * x.abs() + 32 * w * (1 + z1.abs()) * y.abs() for x, y in zip(dz, (c, g * z1))]
        if gated:
            sl.gemm_gated_grad(A, A2, B, "silu", Z1, Z2, G, dA, dA2, dB, opts)
        else:
            sl.gemm_bias_act_grad(1.0, A, B, "silu", Z1, G, dA, dB, db, opts)
            within(D(db), dz[0].sum(1, keepdim=True), (f[0] + 64 * w * dz[0].abs()).sum(1, keepdim=True) +
                   1.1 * u * dz[0].sum(1, keepdim=True).abs())
        for got, x, y in zip((dA, dA2), dz, f):
            want, e = x @ b.t(), (y + 2 * (n + 4) * w * x.abs()) @ b.abs().t()
            within(D(got), want, e + u * (want.abs() + e))
        want = sum(i.t() @ x for i, x in zip((a, a2), dz))
        e = sum(i.abs().t() @ (y + 4 * (m + 4) * w * x.abs()) for i, x, y in zip((a, a2), dz, f))
        within(D(dB), want, e + u * (want.abs() + e))


@pytest.mark.parametrize("p,q", [(2, 1), (2, 2)])
def test_precise_gradient(p, q):
    run_dist(_precise, p * q, p, q, torch.bfloat16)

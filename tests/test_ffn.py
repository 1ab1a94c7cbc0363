"""Fused feed-forward products, their gradients, and gradient clipping against
plain formulas in 64 bits, on the host path and (``gpu``) on the gfx950
kernels.

Tolerances come from the arithmetic.  With u = eps / 2 of the stored type and
w = 2^-24 (2^-53) of the sums', an element of a product over k terms is off by
at most (k + 4) w S, S the sum of the terms' sizes (bias among them), in any
order of the sums; an activation (slope at most 1.13) passes that on and adds
a few w relative to its argument, 16 w (1 + |z|) |z| with the exponential's
error; the store adds u of the value.  Where dZ is rounded between two
products it is off by u + 32 w relative, which the second product's terms
carry."""
import math

import pytest
import torch

import slate_amd as sl
from slate_amd import ops
from slate_amd.core.exceptions import SlateError

DEVS = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
TYPES = [torch.bfloat16, torch.float16, torch.float32, torch.float64]
ACTS = ["identity", "relu", "gelu", "gelu_tanh", "silu"]
HALF = (torch.bfloat16, torch.float16)


def u_of(dt):
    return torch.finfo(dt).eps / 2


def w_of(dt):
    return 2.0 ** -53 if dt == torch.float64 else 2.0 ** -24


def tiny(dt):
    """Half the distance of the smallest subnormal numbers."""
    return torch.finfo(dt).tiny * torch.finfo(dt).eps / 2


def cm(m, n, dt, seed, dev, std=1.0, pad=0, off=0):
    """m x n column-major tensor, leading dimension m + pad, first element off."""
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(n, m, generator=g, dtype=torch.float64) * std).to(dt).to(dev)
    buf = torch.full((off + n * (m + pad),), float("nan"), dtype=dt, device=dev)
    y = buf[off:].view(n, m + pad)[:, :m].t()
    y.copy_(x.t())
    return y


def mat(t, trans=False, nb=64):
    M = sl.Matrix.fromLAPACK(t.shape[0], t.shape[1], t, nb=nb)
    return M.transpose() if trans else M


def act64(name, z):
    if name == "relu":
        return z.clamp(min=0), (z > 0).double()
    if name == "gelu":
        p = 0.5 * torch.special.erfc(-z * math.sqrt(0.5))
        return z * p, p + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        h = torch.tanh(c * (z + 0.044715 * z ** 3))
        return 0.5 * z * (1 + h), 0.5 * (1 + h) + 0.5 * z * (1 - h * h) * c * (1 + 3 * 0.044715 * z * z)
    if name == "silu":
        p = torch.sigmoid(z)
        return z * p, p * (1 + z * (1 - p))
    return z, torch.ones_like(z)


def within(got, want, bound):
    g = got.double()
    bad = ~((g - want).abs() <= bound)
    assert not bad.any(), (int(bad.sum()), float(((g - want).abs() / bound).nan_to_num(1e9).max()))


def act_bound(z, w):
    return 16 * w * (1 + z.abs()) * z.abs()


class Product:
    """Operands, call and oracle of gemm_bias_act."""

    def __init__(self, dt, dev, m, n, k, ta="T", tb="N", bias=1, act="gelu", res=True, keep=True, alpha=0.75, beta=0.5,
                 pad=0, off=0, seed=0, cpad=0):
        self.dt, self.dev, self.m, self.n, self.k, self.act, self.alpha, self.beta = dt, dev, m, n, k, act, alpha, beta
        std = 1 / math.sqrt(max(k, 1))
        self.A = cm(*((k, m) if ta == "T" else (m, k)), dt, seed + 1, dev, std, pad, off)
        self.B = cm(*((n, k) if tb == "T" else (k, n)), dt, seed + 2, dev, 1.0, pad, off)
        self.ta, self.tb = ta, tb
        self.b = None if not bias else (cm(m, 1, dt, seed + 3, dev) if bias == 1 else cm(1, n, dt, seed + 3, dev))
        self.R = cm(m, n, dt, seed + 4, dev, 1.0, pad, off) if res else None
        self.C = cm(m, n, dt, seed + 5, dev, 1.0, cpad, off)
        self.Z = cm(m, n, dt, seed + 6, dev, 1.0, cpad, off) if keep else None

    def handles(self):
        h = [mat(self.A, self.ta == "T"), mat(self.B, self.tb == "T")]
        return h + [None if x is None else mat(x) for x in (self.b, self.R, self.C, self.Z)]

    def want(self):
        a, b = self.A.double(), self.B.double()
        a, b = (a.t() if self.ta == "T" else a).contiguous(), (b.t() if self.tb == "T" else b).contiguous()
        z, S = self.alpha * (a @ b), abs(self.alpha) * (a.abs() @ b.abs())
        if self.b is not None:
            z, S = z + self.b.double(), S + self.b.double().abs()
        w, u = w_of(self.dt), u_of(self.dt)
        ez = (self.k + 4) * w * S + tiny(self.dt)
        y = act64(self.act, z)[0]
        ey = 1.13 * ez + act_bound(z, w)
        if self.R is not None:
            y = y + self.beta * self.R.double()
            ey = ey + 4 * w * (y.abs() + self.beta * self.R.double().abs())
        return z, ez + u * (z.abs() + ez), y, ey + u * (y.abs() + ey)

    def check(self):
        z, ez, y, ey = self.want()
        A, B, b, R, C, Z = self.handles()
        sl.gemm_bias_act(self.alpha, A, B, b, self.act, self.beta, R, C, Z)
        within(self.C, y, ey)
        if self.Z is not None:
            within(self.Z, z, ez)


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("ta,tb", ["TN", "NN", "NT", "TT"])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (64, 1, 128), (40, 5, 72), (131, 67, 203), (96, 130, 16)])
def test_product(dev, dt, ta, tb, m, n, k):
    Product(dt, dev, m, n, k, ta, tb).check()


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("bias", [0, 1, 2])
@pytest.mark.parametrize("res,keep", [(False, False), (True, False), (False, True)])
def test_product_epilogue(dev, dt, act, bias, res, keep):
    Product(dt, dev, 72, 20, 64, act=act, bias=bias, res=res, keep=keep).check()


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("ta,tb", ["TN", "NN", "NT"])
@pytest.mark.parametrize("pad,off,cpad", [(8, 0, 8), (3, 0, 0), (0, 1, 5), (24, 8, 24)])
def test_product_strides(dev, dt, ta, tb, pad, off, cpad):
    """Padded and offset storage: aligned and not; what lies beside it stays."""
    p = Product(dt, dev, 70, 33, 130, ta, tb, pad=pad, off=off, cpad=cpad)
    p.check()
    if cpad:
        assert torch.isnan(p.C.as_strided((cpad, 33), (1, 70 + cpad), p.C.storage_offset() + 70)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("ta,tb", ["TN", "NN", "NT", "TT"])
@pytest.mark.parametrize("m,n,k", [(3601, 3700, 200), (4096, 4096, 256), (1100, 1300, 520), (260, 300, 1000),
                                   (2100, 17, 4100), (513, 16, 8200), (5000, 1, 640), (8, 3000, 72)])
def test_product_sizes(dt, ta, tb, m, n, k):
    """Every tile, whole and ragged, with K in one piece and in several."""
    if dt == torch.float64 and m * n * k > 2e9:
        k = 64 + k % 8
    Product(dt, "cuda", m, n, k, ta, tb, act="silu", alpha=1.0, beta=1.0).check()


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_product_transposed_output(dev, dt):
    p = Product(dt, dev, 66, 41, 80, bias=1)
    z, ez, y, ey = p.want()
    Ct, Zt, Rt = (torch.empty(66, 41, dtype=dt, device=dev).t() for _ in range(3))        # 41 x 66 column-major
    Rt.copy_(p.R.t())
    A, B, b, R, C, Z = p.handles()
    sl.gemm_bias_act(p.alpha, A, B, b, p.act, p.beta, R, mat(Ct, True), mat(Zt, True))
    within(Ct.t(), y, ey)
    within(Zt.t(), z, ez)
    sl.gemm_bias_act(p.alpha, A, B, b, p.act, p.beta, mat(Rt, True), C, mat(Zt, True))
    within(p.C, y, ey)
    within(Zt.t(), z, ez)


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("dt", TYPES)
def test_product_edges(dev, dt):
    nan = float("nan")
    # the residual's own matrix as output
    p = Product(dt, dev, 40, 24, 32, keep=False)
    _, _, y, ey = p.want()
    A, B, b, R, C, _ = p.handles()
    sl.gemm_bias_act(p.alpha, A, B, b, p.act, p.beta, R, R)
    within(p.R, y, ey)
    # beta = 0 reads no residual, alpha = 0 no operand, k = 0 has none
    p = Product(dt, dev, 40, 24, 32, keep=False, beta=0.0)
    p.R.fill_(nan)
    A, B, b, R, C, _ = p.handles()
    sl.gemm_bias_act(p.alpha, A, B, b, p.act, 0.0, R, C)
    assert torch.isfinite(p.C).all()
    p.A.fill_(nan)
    sl.gemm_bias_act(0.0, A, B, b, "identity", 0.0, None, C)
    assert torch.equal(p.C, p.b.expand(40, 24))
    e = torch.empty(0, 40, dtype=dt, device=dev).t()
    f = torch.empty(24, 0, dtype=dt, device=dev).t()
    sl.gemm_bias_act(1.0, mat(e), mat(f), b, "identity", 0.0, None, C)
    assert torch.equal(p.C, p.b.expand(40, 24))
    # no column, no row
    g = torch.empty(0, 32, dtype=dt, device=dev).t()
    h = torch.empty(0, 40, dtype=dt, device=dev).t()
    sl.gemm_bias_act(1.0, A, mat(g), b, "relu", 0.0, None, mat(h))
    # a NaN or an infinity reaches its own column, and no other
    q = Product(dt, dev, 40, 24, 32, keep=False, act="relu", res=False)
    q.B[3, 5] = nan
    q.B[7, 9] = float("inf")
    A, B, b, _, C, _ = q.handles()
    sl.gemm_bias_act(1.0, A, B, b, "relu", 0.0, None, C)
    assert torch.isnan(q.C[:, 5]).all()
    assert (q.C[:, 9].isinf() | (q.C[:, 9] == 0) | q.C[:, 9].isnan()).all()
    rest = [j for j in range(24) if j not in (5, 9)]
    assert torch.isfinite(q.C[:, rest]).all()


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("act", ACTS)
def test_activation_far(dev, dt, act):
    """Far arguments: 0 on the left and z on the right, infinities included, no 0 inf."""
    big = float("inf")
    z = torch.tensor([-big, -6e4, -1e3, -130.0, 0.0, 130.0, 1e3, 6e4, big], dtype=torch.float64)
    one = torch.ones(1, 1, dtype=dt, device=dev)
    Z = z.to(dt).to(dev)[:, None]
    C = torch.empty(1, 9, dtype=dt, device=dev).t()
    sl.gemm_bias_act(0.0, mat(Z), mat(one), mat(Z), act, 0.0, None, mat(C))
    want = Z.double().cpu() if act == "identity" else Z.double().cpu().clamp(min=0)
    # at -130 the largest left tail is silu's, 130 e^-130 = 4.6e-55, which float64 still holds
    assert torch.allclose(C.double().cpu(), want, rtol=0, atol=1e-54)
    D = torch.empty(1, 9, dtype=dt, device=dev).t()
    G = torch.ones(1, 9, dtype=dt, device=dev).t()
    sl.gemm_bias_act_grad(1.0, mat(Z), mat(one), act, mat(Z), mat(G), mat(D), None, None)
    slope = torch.ones(9, 1) if act == "identity" else (Z.cpu() > 0).double()
    keep = [i for i in range(9) if i != 4]
    assert torch.allclose(D.double().cpu()[keep], slope.double()[keep], rtol=0, atol=1e-54)


# ---------------------------------------------------------------- gradients
def grad_call(p, act, which="ABb", bias=1, swap=False, dev_t=lambda t: t):
    """gemm_bias_act_grad on Product p's operands with its Z and R as Z and dC."""
    dt, dev, m, n, k = p.dt, p.dev, p.m, p.n, p.k
    dA = cm(*p.A.shape, dt, 9, dev) if "A" in which else None
    dB = cm(*p.B.shape, dt, 9, dev) if "B" in which else None
    db = (cm(m, 1, dt, 9, dev) if bias == 1 else cm(1, n, dt, 9, dev)) if "b" in which else None
    A, B, _, G, _, Z = p.handles()
    sl.gemm_bias_act_grad(p.alpha, A, B, act, Z, G, None if dA is None else mat(dA, p.ta == "T"),
                          None if dB is None else mat(dB, p.tb == "T"), None if db is None else mat(db))
    a, b, g, z = (x.double() for x in (p.A, p.B, p.R, p.Z))
    a, b = (a.t() if p.ta == "T" else a), (b.t() if p.tb == "T" else b)
    dz = g * act64(act, z)[1]
    u, w = u_of(dt), w_of(dt)
    # a slope is a sum p + z p' of terms of up to 1 + |z|, each off by a few w of
    # itself: the sum passes 0, its error does not, so that it counts relative to
    # the terms; the rounding of dZ to the type counts relative to dZ
    own = 32 * w * (1 + z.abs()) * g.abs() * (act != "identity") + tiny(dt)
    f = own + (0 if act == "identity" else u) * dz.abs()
    al = abs(p.alpha)
    if dA is not None:
        bt = b.t().contiguous()
        want, e = p.alpha * (dz @ bt), al * (f @ bt.abs() + (n + 4) * w * (dz.abs() @ bt.abs())) + tiny(dt)
        within(dA.t() if p.ta == "T" else dA, want, e + u * (want.abs() + e))
    if dB is not None:
        at = a.t().contiguous()
        want, e = p.alpha * (at @ dz), al * (at.abs() @ f + (m + 4) * w * (at.abs() @ dz.abs())) + tiny(dt)
        within(dB.t() if p.tb == "T" else dB, want, e + u * (want.abs() + e))
    if db is not None:
        d = 1 if bias == 1 else 0
        want = dz.sum(d, keepdim=True)
        e = own.sum(d, keepdim=True) + (n if d else m) * w * dz.abs().sum(d, keepdim=True) + tiny(dt)
        within(db, want, e + u * (want.abs() + e))


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("ta,tb", ["TN", "NN", "NT"])
def test_product_grad(dev, dt, act, ta, tb):
    for (m, n, k) in [(1, 1, 1), (48, 1, 40), (70, 33, 50)]:
        grad_call(Product(dt, dev, m, n, k, ta, tb), act)


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("which", ["A", "B", "b", "Bb"])
@pytest.mark.parametrize("bias", [1, 2])
def test_product_grad_parts(dev, dt, which, bias):
    for act in ("identity", "gelu"):
        grad_call(Product(dt, dev, 72, 520, 24, pad=3), act, which, bias)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("m,n,k", [(1503, 777, 1001), (1024, 2048, 512), (4000, 3, 640), (600, 5000, 128)])
def test_product_grad_sizes(dt, m, n, k):
    grad_call(Product(dt, "cuda", m, n, k), "gelu_tanh")


@pytest.mark.parametrize("dev", DEVS)
def test_product_grad_no_tokens(dev):
    """A batch without tokens: zero gradients of weight and bias."""
    dt = torch.bfloat16
    A, dA = cm(32, 16, dt, 1, dev), cm(32, 16, dt, 2, dev)
    B, Z = torch.empty(0, 32, dtype=dt, device=dev).t(), torch.empty(0, 16, dtype=dt, device=dev).t()
    db, dB = cm(16, 1, dt, 3, dev), torch.empty_like(B)
    sl.gemm_bias_act_grad(1.0, mat(A, True), mat(B), "gelu", mat(Z), mat(Z.clone()), mat(dA, True), mat(dB), mat(db))
    assert (dA == 0).all() and (db == 0).all()


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
def test_grad_differences(dev, act):
    """Both backward passes against central differences of the forward calls:
    with h = 1e-4 those are off by h^2 f''' / 6 and 2^-52 f / h, far below 1e-6."""
    dt = torch.float64
    m, n, k, h = 12, 7, 9, 1e-4
    t = {x: cm(*s, dt, i, dev) for i, (x, s) in enumerate(dict(
        A=(k, m), A2=(k, m), B=(k, n), b=(m, 1), G=(m, n), R=(m, n)).items())}
    C, Z1, Z2 = (cm(m, n, dt, 50 + i, dev) for i in range(3))
    M = {x: mat(v, x in ("A", "A2")) for x, v in t.items()}

    def plain():
        sl.gemm_bias_act(0.7, M["A"], M["B"], M["b"], act, 0.5, M["R"], mat(C), mat(Z1))
        return float((C * t["G"]).sum())

    def gated():
        sl.gemm_gated(M["A"], M["A2"], M["B"], act, mat(C), mat(Z1), mat(Z2))
        return float((C * t["G"]).sum())

    def slope(f, x, i, j):
        v = float(t[x][i, j])
        t[x][i, j] = v + h
        up = f()
        t[x][i, j] = v - h
        down = f()
        t[x][i, j] = v
        return (up - down) / (2 * h)

    d = {x: cm(*t[x].shape, dt, 60, dev) for x in ("A", "A2", "B", "b")}
    plain()
    sl.gemm_bias_act_grad(0.7, M["A"], M["B"], act, mat(Z1), M["G"], mat(d["A"], True), mat(d["B"]), mat(d["b"]))
    for x in ("A", "B", "b"):
        for (i, j) in [(0, 0), (t[x].shape[0] - 1, t[x].shape[1] - 1), (t[x].shape[0] // 2, 0)]:
            assert abs(slope(plain, x, i, j) - float(d[x][i, j])) < 1e-6
    gated()
    sl.gemm_gated_grad(M["A"], M["A2"], M["B"], act, mat(Z1), mat(Z2), M["G"], mat(d["A"], True), mat(d["A2"], True),
                       mat(d["B"]))
    for x in ("A", "A2", "B"):
        for (i, j) in [(0, 0), (t[x].shape[0] - 1, t[x].shape[1] - 1), (t[x].shape[0] // 2, 0)]:
            assert abs(slope(gated, x, i, j) - float(d[x][i, j])) < 1e-6


# -------------------------------------------------------------------- gated
class Gated:
    def __init__(self, dt, dev, m, n, k, ta="T", tb="N", act="silu", pad=0, off=0):
        self.dt, self.dev, self.m, self.n, self.k, self.ta, self.tb, self.act = dt, dev, m, n, k, ta, tb, act
        std = 1 / math.sqrt(max(k, 1))
        shape = (k, m) if ta == "T" else (m, k)
        self.A1, self.A2 = cm(*shape, dt, 1, dev, std, pad, off), cm(*shape, dt, 2, dev, std, pad, off)
        self.B = cm(*((n, k) if tb == "T" else (k, n)), dt, 3, dev, 1.0, pad, off)
        self.C, self.Z1, self.Z2 = (cm(m, n, dt, 4 + i, dev, 1.0, pad, off) for i in range(3))
        self.G = cm(m, n, dt, 7, dev, 1.0, pad, off)

    def dense(self):
        a1, a2, b = self.A1.double(), self.A2.double(), self.B.double()
        if self.ta == "T":
            a1, a2 = a1.t().contiguous(), a2.t().contiguous()
        return a1, a2, (b.t().contiguous() if self.tb == "T" else b)

    def handles(self):
        return [mat(self.A1, self.ta == "T"), mat(self.A2, self.ta == "T"), mat(self.B, self.tb == "T")]

    def want(self):
        a1, a2, b = self.dense()
        w, u = w_of(self.dt), u_of(self.dt)
        z1, z2 = a1 @ b, a2 @ b
        e1, e2 = ((self.k + 4) * w * (a.abs() @ b.abs()) + tiny(self.dt) for a in (a1, a2))
        v = act64(self.act, z1)[0]
        ev = 1.13 * e1 + act_bound(z1, w)
        y = v * z2
        ey = ev * z2.abs() + e2 * v.abs() + ev * e2 + 2 * w * y.abs() + tiny(self.dt)
        return [(z1, e1 + u * (z1.abs() + e1)), (z2, e2 + u * (z2.abs() + e2)), (y, ey + u * (y.abs() + ey))]

    def check(self):
        (z1, e1), (z2, e2), (y, ey) = self.want()
        sl.gemm_gated(*self.handles(), self.act, mat(self.C), mat(self.Z1), mat(self.Z2))
        within(self.C, y, ey)
        within(self.Z1, z1, e1)
        within(self.Z2, z2, e2)
        self.C.fill_(0)
        sl.gemm_gated(*self.handles(), self.act, mat(self.C))
        within(self.C, y, ey)

    def check_grad(self, which=("A1", "A2", "B")):
        dt, u, w = self.dt, u_of(self.dt), w_of(self.dt)
        a1, a2, b = self.dense()
        z1, z2, g = self.Z1.double(), self.Z2.double(), self.G.double()
        d = {x: cm(*getattr(self, x).shape, dt, 9, self.dev) if x in which else None for x in ("A1", "A2", "B")}
        t = {"A1": self.ta == "T", "A2": self.ta == "T", "B": self.tb == "T"}
        sl.gemm_gated_grad(*self.handles(), self.act, mat(self.Z1), mat(self.Z2), mat(self.G),
                           *(None if d[x] is None else mat(d[x], t[x]) for x in ("A1", "A2", "B")))
        v, s = act64(self.act, z1)
        d1, d2 = g * z2 * s, g * v
        one = u + 32 * w * (1 + z1.abs().max())
        bt = b.t().contiguous()
        # a slope's own error is relative to 1, not to itself (it passes 0)
        f1, f2 = one * d1.abs() + 32 * w * (g * z2).abs() + tiny(dt), one * d2.abs() + 32 * w * (g * z1).abs() + tiny(dt)
        wants = {"A1": (d1 @ bt, f1 @ bt.abs() + (self.n + 4) * w * (d1.abs() @ bt.abs())),
                 "A2": (d2 @ bt, f2 @ bt.abs() + (self.n + 4) * w * (d2.abs() @ bt.abs())),
                 "B": (a1.t().contiguous() @ d1 + a2.t().contiguous() @ d2,
                       sum(a.abs().t().contiguous() @ f + (2 * self.m + 4) * w * (a.abs().t().contiguous() @ x.abs())
                           for a, x, f in ((a1, d1, f1), (a2, d2, f2))))}
        for x in which:
            want, e = wants[x]
            e = e + tiny(dt)
            within(d[x].t() if t[x] else d[x], want, e + u * (want.abs() + e))


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("ta,tb", ["TN", "NN", "NT", "TT"])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (64, 1, 128), (131, 67, 75)])
def test_gated(dev, dt, ta, tb, m, n, k):
    Gated(dt, dev, m, n, k, ta, tb).check()


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("pad,off", [(0, 0), (8, 8), (3, 1)])
def test_gated_strides(dev, dt, act, pad, off):
    g = Gated(dt, dev, 70, 33, 66, act=act, pad=pad, off=off)
    g.check_grad()
    g.check()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("ta,tb", ["TN", "NN"])
@pytest.mark.parametrize("m,n,k", [(1801, 3700, 200), (2048, 4096, 256), (700, 1300, 520), (2100, 17, 4100), (5000, 1, 640)])
def test_gated_sizes(dt, ta, tb, m, n, k):
    Gated(dt, "cuda", m, n, k, ta, tb).check()


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("ta,tb", ["TN", "NN", "NT"])
def test_gated_grad(dev, dt, ta, tb):
    for (m, n, k) in [(1, 1, 1), (48, 1, 40), (70, 33, 50)]:
        Gated(dt, dev, m, n, k, ta, tb).check_grad()
    for which in (("A1",), ("A2",), ("B",), ("A1", "B")):
        Gated(dt, dev, 33, 20, 40, ta, tb).check_grad(which)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("m,n,k", [(1503, 777, 500), (1024, 2048, 512), (2560, 515, 1024), (3000, 2, 640)])
def test_gated_grad_sizes(dt, m, n, k):
    Gated(dt, "cuda", m, n, k, act="gelu").check_grad()


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("dt", [torch.float16, torch.float32])
def test_gated_mixed_orientation(dev, dt):
    """Operands, outputs and stored products of either orientation."""
    g = Gated(dt, dev, 40, 24, 32)
    (z1, e1), (z2, e2), (y, ey) = g.want()
    turn = lambda x: torch.empty(x.shape[0], x.shape[1], dtype=dt, device=dev).t()      # noqa: E731
    Ct, Z1t, A2t = turn(g.C), turn(g.Z1), turn(g.A2)
    A2t.copy_(g.A2.t())
    A1, A2, B = g.handles()
    sl.gemm_gated(A1, mat(A2t), B, g.act, mat(Ct, True), mat(Z1t, True), mat(g.Z2))
    within(Ct.t(), y, ey)
    within(Z1t.t(), z1, e1)
    within(g.Z2, z2, e2)
    # the backward pass from a transposed Z1 is that from Z1
    g.Z1.copy_(Z1t.t())
    d = [[torch.empty_like(x) for x in (g.A1, g.A2, g.B)] for _ in range(2)]
    for k, (z, a2) in enumerate(((mat(Z1t, True), mat(A2t)), (mat(g.Z1), A2))):
        sl.gemm_gated_grad(A1, a2, B, g.act, z, mat(g.Z2), mat(g.G), mat(d[k][0], True), mat(d[k][1], True), mat(d[k][2]))
    for x, v in zip(*d):
        assert torch.equal(x, v)


# ----------------------------------------------------------------- clipping
def clip_case(dt, dev, shapes, std=0.02, pad=0, off=0):
    return [cm(m, n, dt, 100 + i, dev, std, pad, off) for i, (m, n) in enumerate(shapes)]


def clip_want(xs, limit):
    wide = lambda x: torch.view_as_real(x.contiguous()).double() if x.is_complex() else x.double()      # noqa: E731
    s = math.sqrt(math.fsum(float((wide(x) ** 2).sum()) for x in xs))
    return s, min(1.0, limit / s) if s else 1.0


CLIP_TYPES = [(torch.bfloat16,) * 2, (torch.bfloat16, torch.float32), (torch.float16,) * 2, (torch.float16, torch.float32),
              (torch.float32,) * 2, (torch.float64,) * 2, (torch.complex64,) * 2, (torch.complex128,) * 2]


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("dt,out", CLIP_TYPES)
@pytest.mark.parametrize("pad,off", [(0, 0), (3, 1), (8, 0)])
@pytest.mark.parametrize("limit", [0.25, 1e6, 0.0])
def test_clip(dev, dt, out, pad, off, limit):
    if dt.is_complex:
        mk = lambda i, m, n: torch.complex(cm(m, n, dt.to_real(), i, dev, .02), cm(m, n, dt.to_real(), i + 50, dev, .02))  # noqa: E731
        xs = [mk(i, m, n).t().contiguous().t() for i, (m, n) in enumerate([(30, 20), (1, 7), (200, 1)])]
    else:
        xs = clip_case(dt, dev, [(300, 200), (1, 17), (65, 1), (33, 130), (1, 1)], pad=pad, off=off)
    ys = [cm(*x.shape, out.to_real() if out.is_complex else out, 1, dev, 1.0, pad) for x in xs]
    if out.is_complex:
        ys = [torch.zeros_like(x) for x in xs]
    s, f = clip_want(xs, limit)
    got = sl.clip_norm(limit, [mat(x) for x in xs], [mat(y) for y in ys])
    n = sum(x.numel() for x in xs)
    assert got.dtype == torch.float64 and abs(float(got) - s) <= (n + 4) * 2.0 ** -53 * s
    # the factor is rounded to the sums' type, the product again, then the store
    rt = out.to_real() if out.is_complex else out
    rel = u_of(rt) + 3 * w_of(rt) + (n + 4) * 2.0 ** -53
    for x, y in zip(xs, ys):
        a, b = (torch.view_as_real(v.contiguous()).double() if v.is_complex() else v.double() for v in (x, y))
        assert ((b - a * f).abs() <= rel * (a * f).abs() + tiny(rt)).all()
        if limit == 1e6 and dt == out:
            assert torch.equal(x, y)
    # in place, the same values
    if dt == out:
        sl.clip_norm(limit, [mat(x) for x in xs])
        for x, y in zip(xs, ys):
            assert torch.equal(x, y)
            if pad and x.shape[1] > 1 and not dt.is_complex:
                m = x.shape[0]
                assert torch.isnan(x.as_strided((pad, x.shape[1]), (1, m + pad), x.storage_offset() + m)).all()


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("count", [0, 1, 48, 49, 200])
def test_clip_many(dev, count):
    """More matrices than one launch describes, empty ones among them."""
    xs = clip_case(torch.float32, dev, [((7 * i) % 23 if i % 9 else 0, 1 + i % 11) for i in range(count)], 1.0)
    s, f = clip_want(xs, 2.0)
    want = [x.double() * f for x in xs]
    got = sl.clip_norm(2.0, [mat(x) for x in xs])
    assert abs(float(got) - s) <= 1e-12 * max(s, 1)
    for x, w in zip(xs, want):
        assert ((x.double() - w).abs() <= 2.0 ** -22 * w.abs()).all()
    assert abs(sl.global_norm([mat(x) for x in xs]) - min(s, 2.0)) <= 1e-6 * max(1, s)


@pytest.mark.parametrize("dev", DEVS)
def test_clip_extremes(dev):
    """Squares outside a type's range, and norms that are not finite."""
    for dt, v in ((torch.float32, 1e30), (torch.float32, 1e-30), (torch.float64, 1e300), (torch.float64, 1e-300),
                  (torch.float64, 1e140), (torch.float64, 5e-324)):
        x = torch.full((1000,), v, dtype=dt, device=dev)[:, None]
        want = float(x[0, 0]) * math.sqrt(1000)
        assert abs(sl.global_norm([mat(x)]) - want) <= 1e-12 * want
    x = torch.tensor([3e200, 4e200, 1.0, 1e-200], dtype=torch.float64, device=dev)[:, None]
    assert abs(sl.global_norm([mat(x)]) - 5e200) <= 1e188
    x = torch.tensor([3e-170, 4e-170, 1e-300], dtype=torch.float64, device=dev)[:, None]
    assert abs(sl.global_norm([mat(x)]) - 5e-170) <= 1e-182
    for bad in (float("inf"), float("nan")):
        for dt in (torch.float32, torch.bfloat16, torch.float64):
            x = cm(64, 40, dt, 1, dev)
            x[5, 6] = bad
            y, z = x.clone(), cm(64, 40, dt, 2, dev)
            s = float(sl.clip_norm(1.0, [mat(x)]))
            assert (s != s) if bad != bad else s == bad
            assert torch.equal(x.view(torch.uint8) if False else x.nan_to_num(7.0), y.nan_to_num(7.0))
            sl.clip_norm(1.0, [mat(x)], [mat(z)])
            assert torch.equal(z.nan_to_num(7.0), y.nan_to_num(7.0))
    z = torch.zeros(16, 16, device=dev).t()
    assert float(sl.clip_norm(0.0, [mat(z)])) == 0.0 and (z == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32, torch.float64])
def test_clip_sizes(dt):
    xs = clip_case(dt, "cuda", [(4096, 1024), (4099, 513), (100003, 1), (5, 50000)])
    s, f = clip_want(xs, 1.0)
    want = [x.double() * f for x in xs]
    got = sl.clip_norm(1.0, [mat(x) for x in xs])
    assert abs(float(got) - s) <= 1e-9 * s
    for x, w in zip(xs, want):
        assert ((x.double() - w).abs() <= (u_of(dt) + 4 * w_of(dt) + 1e-9 * (dt == torch.float64)) * w.abs() + tiny(dt)).all()


# ------------------------------------------------------------------- copies
@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("src", TYPES)
@pytest.mark.parametrize("dst", TYPES)
@pytest.mark.parametrize("trans", "NT")
def test_copy_half(dev, src, dst, trans):
    """Precision conversion of sl.copy to and from the 16-bit types, ties to even."""
    if src not in HALF and dst not in HALF:
        pytest.skip("the other kernels")
    x = cm(67, 45, src, 3, dev)
    x[0, :6] = torch.tensor([1 + 2.0 ** -9, 1 + 3 * 2.0 ** -9, 1 + 2.0 ** -12, 65519.0, 1e-7, -0.0], dtype=torch.float64).to(src)
    y = cm(*((67, 45) if trans == "N" else (45, 67)), dst, 4, dev)
    ops.gecopy(x, y, trans=trans)
    want = x if trans == "N" else x.t()
    assert torch.equal(y.cpu(), want.cpu().to(dst))
    if trans == "N":
        A, B = mat(x), mat(cm(67, 45, dst, 5, dev))
        sl.copy(A, B)
        assert torch.equal(B.to_dense().cpu(), x.cpu().to(dst))


# ----------------------------------------------------------------- refusals
@pytest.mark.parametrize("dev", DEVS)
def test_refusals(dev):
    f = torch.float32
    A, B, C = (mat(cm(m, n, f, 1, dev)) for (m, n) in ((16, 8), (8, 12), (16, 12)))
    b, R = mat(cm(16, 1, f, 2, dev)), mat(cm(16, 12, f, 3, dev))
    ok = lambda **k: sl.gemm_bias_act(*[{**dict(alpha=1.0, A=A, B=B, bias=b, act="relu", beta=1.0, R=R, C=C), **k}[x]  # noqa: E731
                                        for x in ("alpha", "A", "B", "bias", "act", "beta", "R", "C")])
    ok()
    for bad in (dict(A=mat(cm(16, 9, f, 1, dev))), dict(B=mat(cm(8, 11, f, 1, dev))), dict(R=mat(cm(16, 11, f, 1, dev))),
                dict(bias=mat(cm(12, 1, f, 1, dev))), dict(bias=mat(cm(16, 2, f, 1, dev))), dict(act="tanh"), dict(act=None),
                dict(A=mat(cm(16, 8, torch.float64, 1, dev))), dict(R=mat(cm(16, 12, torch.bfloat16, 1, dev))),
                dict(C=A), dict(R=C.transpose())):
        with pytest.raises(SlateError):
            ok(**bad)
    with pytest.raises(SlateError):
        sl.gemm_bias_act(1.0, A, B, b, "relu", 1.0, R, C, C)
    square = mat(cm(8, 8, f, 1, dev))
    for call in (lambda: sl.gemm_bias_act(1.0, square, square, None, "relu", 0.0, None, square),
                 lambda: sl.gemm_gated(square, square, square, "relu", square),
                 lambda: sl.gemm_gated(A, A, B, "relu", C, R, R),
                 lambda: sl.gemm_gated_grad(A, A, B, "relu", None, R, C, None, None, None),
                 lambda: sl.gemm_bias_act_grad(1.0, A, B, "relu", None, C, mat(cm(16, 8, f, 1, dev)), None, None),
                 lambda: sl.gemm_bias_act_grad(1.0, A, B, "relu", R, C, A, None, None)):
        with pytest.raises(SlateError):
            call()
    z = [mat(torch.zeros(4, 4, dtype=torch.complex64, device=dev).t()) for _ in range(3)]
    with pytest.raises(SlateError):
        sl.gemm_bias_act(1.0, z[0], z[1], None, "relu", 0.0, None, z[2])
    H = sl.HermitianMatrix.fromLAPACK(sl.Uplo.Lower, 8, cm(8, 8, f, 1, dev))
    with pytest.raises(SlateError):
        sl.gemm_bias_act(1.0, H, square, None, "relu", 0.0, None, mat(cm(8, 8, f, 2, dev)))
    spread = torch.zeros(8, 1, dtype=f, device=dev).expand(8, 4)
    with pytest.raises(SlateError):
        sl.gemm_bias_act(1.0, square, sl.Matrix.fromLAPACK(8, 4, spread.as_strided((8, 4), (1, 0)), nb=8), None, "relu", 0.0,
                         None, mat(cm(8, 4, f, 2, dev)))
    for call in (lambda: sl.clip_norm(-1.0, [A]), lambda: sl.clip_norm(float("nan"), [A]), lambda: sl.clip_norm(1.0, A),
                 lambda: sl.clip_norm(1.0, [A, A]), lambda: sl.clip_norm(1.0, [A, B], [A]),
                 lambda: sl.clip_norm(1.0, [A], [B]), lambda: sl.clip_norm(1.0, [A, mat(cm(4, 4, torch.float64, 1, dev))]),
                 lambda: sl.clip_norm(1.0, [mat(cm(4, 4, torch.float64, 1, dev))], [mat(cm(4, 4, f, 1, dev))]),
                 lambda: sl.clip_norm(1.0, [H]), lambda: sl.clip_norm(1.0, [A], [B.transpose()])):
        with pytest.raises(SlateError):
            call()


@pytest.mark.parametrize("dev", DEVS)
def test_blocks_of_one_matrix(dev):
    """Disjoint blocks of one storage are operands and outputs of one call."""
    big = torch.zeros(40, 64, dtype=torch.float32, device=dev).t()
    big.copy_(torch.randn(64, 40, generator=torch.Generator().manual_seed(1)).to(dev))
    M = sl.Matrix.fromLAPACK(64, 40, big, nb=8)
    A, B, C = M.slice(0, 31, 0, 15), M.slice(32, 47, 0, 23), M.slice(32, 63, 16, 39)
    with pytest.raises(SlateError):                      # B's columns 16.. lie in C
        sl.gemm_bias_act(1.0, A, B, None, "relu", 0.0, None, C)
    B = M.slice(0, 15, 16, 39)
    keep = big.clone()
    sl.gemm_bias_act(1.0, A, B, None, "relu", 0.0, None, C)
    want = (keep[:32, :16].double() @ keep[:16, 16:].double()).clamp(min=0)
    S = keep[:32, :16].double().abs() @ keep[:16, 16:].double().abs()
    within(big[32:, 16:], want, 24 * 2.0 ** -24 * S + 2.0 ** -24 * want)
    assert torch.equal(big[:32], keep[:32]) and torch.equal(big[32:, :16], keep[32:, :16])


# ------------------------------------------------------------------ together
def block(dt, dev, t=45, d=72, f=104, seed=0):
    """One feed-forward block's step: gated projection, projection back onto
    the residual, both backward passes, and the clipping of all gradients."""
    s = dict(x=cm(d, t, dt, seed + 1, dev), wg=cm(d, f, dt, seed + 2, dev, d ** -.5), wu=cm(d, f, dt, seed + 3, dev, d ** -.5),
             wd=cm(f, d, dt, seed + 4, dev, f ** -.5), b=cm(d, 1, dt, seed + 5, dev), g=cm(d, t, dt, seed + 6, dev))
    for n, (a, b) in dict(h=(f, t), z1=(f, t), z2=(f, t), y=(d, t), dh=(f, t), dx=(d, t)).items():
        s[n] = cm(a, b, dt, 20, dev)
    for n in ("wg", "wu", "wd", "b"):
        s["d" + n] = torch.empty_like(s[n])
    H = {n: mat(v, n in ("wg", "wu", "wd", "dwg", "dwu", "dwd")) for n, v in s.items()}

    def step():
        sl.gemm_gated(H["wg"], H["wu"], H["x"], "silu", H["h"], H["z1"], H["z2"])
        sl.gemm_bias_act(1.0, H["wd"], H["h"], H["b"], "identity", 1.0, H["x"], H["y"])
        sl.gemm_bias_act_grad(1.0, H["wd"], H["h"], "identity", None, H["g"], H["dwd"], H["dh"], H["db"])
        sl.gemm_gated_grad(H["wg"], H["wu"], H["x"], "silu", H["z1"], H["z2"], H["dh"], H["dwg"], H["dwu"], H["dx"])
        return sl.clip_norm(0.5, [H[n] for n in ("dwg", "dwu", "dwd", "db")])

    return s, step


OUT = ("y", "dx", "dwg", "dwu", "dwd", "db")


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("dt", TYPES)
def test_block(dev, dt):
    s, step = block(dt, dev)
    norm = step()
    v = {n: x.double().detach().clone().requires_grad_(n in ("x", "wg", "wu", "wd", "b"))
         for n, x in s.items() if n in ("x", "wg", "wu", "wd", "b", "g")}
    x = v["x"]
    h = torch.nn.functional.silu(v["wg"].t() @ x) * (v["wu"].t() @ x)
    y = v["wd"].t() @ h + v["b"] + x
    (y * v["g"]).sum().backward()
    want = dict(y=y.detach(), dwg=v["wg"].grad, dwu=v["wu"].grad, dwd=v["wd"].grad, db=v["b"].grad, dx=x.grad - v["g"])
    total = math.sqrt(sum(float((want[n] ** 2).sum()) for n in ("dwg", "dwu", "dwd", "db")))
    # at most six roundings to the type (h, z1, z2, dh, dz, the gradient) and the
    # sums' own errors lie on a path, each of relative 2-norm at most u (w (k + 4))
    tol = 8 * u_of(dt) + 8 * (104 + 4) * w_of(dt)
    assert abs(float(norm) - total) <= tol * total
    for n in OUT:
        ref = want[n] * (min(1, 0.5 / total) if n in ("dwg", "dwu", "dwd", "db") else 1)
        assert float((s[n].double() - ref).norm()) <= 2 * tol * float(ref.norm()), n


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_block_stream_and_repeat(dt):
    """Another stream, and the same bits on every run."""
    s, step = block(dt, "cuda", 300, 256, 520)
    n0 = step()
    first = {n: s[n].clone() for n in OUT}
    side = torch.cuda.Stream()
    for n in OUT:
        s[n].fill_(0)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        n1 = step()
    torch.cuda.current_stream().wait_stream(side)
    assert float(n0) == float(n1)
    for n in OUT:
        assert torch.equal(s[n], first[n]), n


@pytest.mark.gpu
def test_block_two_streams():
    """Two steps at once on two streams, each with its own workspaces."""
    a, b = block(torch.bfloat16, "cuda", 300, 256, 520), block(torch.bfloat16, "cuda", 300, 256, 520, seed=40)
    want = []
    for s, step in (a, b):
        step()
        want.append({n: s[n].clone() for n in OUT})
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for (s, step), st in zip((a, b), sides):
            with torch.cuda.stream(st):
                step()
    torch.cuda.synchronize()
    for (s, _), w in zip((a, b), want):
        for n in OUT:
            assert torch.equal(s[n], w[n]), n


@pytest.mark.gpu
def test_block_graphs():
    """Two captured steps that share a pool, replayed with eager work between."""
    a, b = block(torch.bfloat16, "cuda", 1, 256, 520), block(torch.bfloat16, "cuda", 77, 256, 520, seed=40)
    want = []
    for s, step in (a, b):
        step()
        want.append({n: s[n].clone() for n in OUT})
    torch.cuda.synchronize()
    graphs, pool = [], torch.cuda.graph_pool_handle()
    for s, step in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            step()
        graphs.append(g)
    for _ in range(3):
        for (s, step), g, w in zip((a, b), graphs, want):
            for n in OUT:
                s[n].fill_(float("nan"))
            g.replay()
            torch.cuda.synchronize()
            for n in OUT:
                assert torch.equal(s[n], w[n]), n
        a[1]()
        torch.cuda.synchronize()


@pytest.mark.gpu
def test_no_host_sync():
    s, step = block(torch.bfloat16, "cuda", 300, 256, 520)
    step()
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        step()
    finally:
        torch.cuda.set_sync_debug_mode("default")


@pytest.mark.gpu
@pytest.mark.parametrize("dt", HALF)
@pytest.mark.parametrize("ta,tb", ["TN", "NN", "NT", "TT"])
@pytest.mark.parametrize("m,n,k", [(4090, 260, 4000), (1020, 2040, 1500), (1030, 250, 8200), (2000, 4100, 1000),
                                   (1640, 4040, 5000), (8190, 510, 300), (200, 130, 5000), (70, 40, 65)])
def test_half_tiles(dt, ta, tb, m, n, k):
    """16-bit tiles of 64, 128 and 256 rows, two and three slots, with K in one piece and in several."""
    Product(dt, "cuda", m, n, k, ta, tb, act="gelu", pad=-m % 8 if ta == "N" else -k % 8).check()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", HALF)
@pytest.mark.parametrize("ta,tb", ["TN", "NN", "NT", "TT"])
@pytest.mark.parametrize("pad,off", [(0, 0), (3, 1)])
def test_half_unaligned(dt, ta, tb, pad, off):
    """Large operands whose columns lie across 16 bytes; what lies between the columns (NaN) is not used."""
    Product(dt, "cuda", 2053, 2049, 2051, ta, tb, act="silu", pad=pad, off=off).check()
    Gated(dt, "cuda", 1101, 2051, 2053, ta, tb, pad=pad, off=off).check()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", HALF)
@pytest.mark.parametrize("ta,tb", ["TN", "NN"])
def test_half_unaligned_grad(dt, ta, tb):
    grad_call(Product(dt, "cuda", 2051, 2049, 2053, ta, tb, pad=3), "gelu")
    Gated(dt, "cuda", 1103, 2049, 2051, ta, tb, pad=1, off=3).check_grad()


@pytest.mark.parametrize("dev", DEVS)
def test_clip_overlaps(dev):
    """Matrices that are written share no element with others; blocks of one buffer may lie in each other's range."""
    x = cm(40, 30, torch.float32, 1, dev)
    y = cm(40, 30, torch.float32, 2, dev)
    norm, f = clip_want([x[:20], x[20:]], 1.0)
    was = x.double()
    halves = [mat(x[:20]), mat(x[20:])]
    for A, B in (([mat(x), mat(x)], None), ([mat(x), mat(x[5:9])], None), ([mat(x[:21]), mat(x[20:])], None),
                 (halves, [mat(y[:20]), mat(x[:20])]), ([mat(x[:20])], [mat(x[1:21])]), (halves[:1] * 2, [mat(y[:20])] * 2)):
        with pytest.raises(SlateError, match="overlap"):
            sl.clip_norm(1.0, A, B)
    # read twice, written once each
    s = sl.clip_norm(1e9, halves[:1] * 2, [mat(y[:20]), mat(y[20:])])
    assert torch.equal(y[:20], x[:20]) and torch.equal(y[20:], x[:20])
    assert abs(float(s) - math.sqrt(2) * float(x[:20].double().norm())) < 1e-6
    s = sl.clip_norm(1.0, halves)
    assert abs(float(s) - norm) <= 1e-12 * norm
    within(x, f * was, 4 * 2.0 ** -24 * f * was.abs())


@pytest.mark.gpu
def test_far_offsets():
    """Elements more than 2^31 beyond the first: many columns, and long sums in both layouts."""
    n = 2 ** 25 + 3
    A = cm(72, 40, torch.bfloat16, 1, "cuda", 0.1)
    B = torch.zeros(n, 72, dtype=torch.bfloat16, device="cuda")
    at = torch.tensor([0, n // 2, n - 65, n - 1], device="cuda")
    B[at] = torch.randn(4, 72, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).cuda()
    C = torch.full((n, 40), 7.0, dtype=torch.bfloat16, device="cuda")
    sl.gemm_bias_act(1.0, mat(A, True, 2 ** 20), mat(B.t(), nb=2 ** 20), None, "silu", 0.0, None, mat(C.t(), nb=2 ** 20))
    a, b = A.double(), B[at].double()
    z, S = b @ a, b.abs() @ a.abs()
    y = act64("silu", z)[0]
    e = 1.13 * 76 * 2.0 ** -24 * S + act_bound(z, 2.0 ** -24)
    within(C[at], y, e + 2.0 ** -8 * (y.abs() + e))
    C[at] = 0
    assert int(torch.count_nonzero(C)) == 0
    del B, C
    # sums of few terms, exact in 16 bits: 8 rows of 2^28 + 64 elements, and 2^25 + 5 columns of 72
    for rows, k, trans in ((8, 2 ** 28 + 64, True), (72, 2 ** 25 + 5, False)):
        X = torch.zeros((rows, k) if trans else (k, rows), dtype=torch.bfloat16, device="cuda")
        Y = torch.zeros(2, k, dtype=torch.bfloat16, device="cuda")
        for i, p in enumerate((0, k // 2, k - 1)):
            (X[:, p] if trans else X[p]).copy_(torch.arange(1, rows + 1, device="cuda") * 2.0 ** i / 8)
            Y[:, p] = torch.tensor([1.0, 2.0], device="cuda")
        C = torch.empty(2, rows, dtype=torch.float32, device="cuda").to(torch.bfloat16)
        sl.gemm_bias_act(1.0, mat(X.t(), trans, 2 ** 28), mat(Y.t(), nb=2 ** 28), None, "identity", 0.0, None, mat(C.t()))
        want = torch.arange(1, rows + 1).double() * 7 / 8
        want = torch.stack([want, 2 * want])
        within(C.cpu(), want, 2.0 ** -8 * want.abs())
        del X, Y


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("ta,tb", ["TN", "NN", "NT", "TT"])
@pytest.mark.parametrize("pad,off", [(0, 0), (1, 1)])
def test_short_columns(dev, dt, ta, tb, pad, off):
    """Columns of fewer than 16 bytes, aligned and not."""
    for m, n, k in ((5, 40, 3), (3, 70, 6), (90, 5, 7), (7, 33, 70), (70, 1, 1), (1, 20, 9)):
        Product(dt, dev, m, n, k, ta, tb, pad=pad, off=off).check()
    Gated(dt, dev, 6, 35, 5, ta, tb, pad=pad, off=off).check()
    Gated(dt, dev, 6, 35, 5, ta, tb, pad=pad, off=off).check_grad()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("m,n,k", [(70, 40, 130), (40, 20, 3), (3, 90, 70)])
def test_wide_leading_dimension(dt, m, n, k):
    """Columns so far apart that 32 bits do not reach over a tile."""
    es = torch.finfo(dt).bits // 8
    far = 2 ** 31 // 256 // es + 5                        # along k; columns across it in the second call
    for ta, far in (("T", far), ("N", min(2 ** 24, 2 ** 32 // (k * es)) + 3)):
        p = Product(dt, "cuda", m, n, k, ta, "N")
        rows, cols = p.A.shape
        buf = torch.full((cols * far,), float("nan"), dtype=dt, device="cuda")
        A = buf.as_strided((rows, cols), (1, far))
        A.copy_(p.A)
        p.A = A
        p.check()
        del buf, A


@pytest.mark.gpu
@pytest.mark.parametrize("dt", HALF)
@pytest.mark.parametrize("ta,tb", ["TN", "NN", "NT", "TT"])
def test_short_last_step(dt, ta, tb):
    """K that ends early in its last step, of one product and of a sum of two; the same bits every time."""
    for k in (72, 136, 200, 328, 520):
        p = Product(dt, "cuda", 328, 264, k, ta, tb)
        p.check()
        first = p.C.clone()
        for _ in range(8):
            sl.gemm_bias_act(p.alpha, *p.handles()[:3], p.act, p.beta, *p.handles()[3:])
            assert torch.equal(p.C, first)
        Gated(dt, "cuda", k, 264, 328, ta, tb).check_grad(("B",))


def other_kinds(A):
    """Views of a square general matrix whose elements are not all its own."""
    up = sl.Uplo.Upper
    return [sl.HermitianMatrix(sl.Uplo.Lower, A), sl.SymmetricMatrix(up, A), sl.TrapezoidMatrix(up, matrix=A),
            sl.TriangularMatrix(sl.Uplo.Lower, sl.Diag.NonUnit, A), sl.BandMatrix(kl=1, ku=2, matrix=A),
            sl.TriangularBandMatrix(sl.Uplo.Lower, kd=2, matrix=A), sl.HermitianBandMatrix(sl.Uplo.Lower, kd=2, matrix=A)]


@pytest.mark.parametrize("dev", DEVS)
def test_other_kinds_refused(dev):
    """Hermitian, triangular and band views are refused whether or not the
    matrix they were made of has been an operand before."""
    x = cm(8, 8, torch.float32, 1, dev)
    was = x.clone()
    for used in (False, True):
        A = mat(x, nb=4)
        if used:
            sl.global_norm([A])
        for H in other_kinds(A):
            for call in (lambda: sl.global_norm([H]), lambda: sl.clip_norm(1e-3, [H]), lambda: sl.clip_norm(1e-3, [A], [H]),
                         lambda: sl.gemm_bias_act(1.0, H, A, None, "relu", 0.0, None, mat(cm(8, 8, torch.float32, 2, dev))),
                         lambda: sl.gemm_gated(H, A, mat(x), "relu", mat(cm(8, 8, torch.float32, 2, dev)))):
                with pytest.raises(SlateError):
                    call()
            with pytest.raises(SlateError):
                sl.global_norm([H])                          # and the second time
    assert torch.equal(x, was)


def test_operand_of_another_storage():
    """A view that is given another storage has that one's operand."""
    x, y = (cm(8, 8, torch.float32, i, "cpu") for i in (1, 2))
    A, B = mat(x), mat(y)
    sl.global_norm([A])
    A.storage = B.storage
    assert abs(sl.global_norm([A]) - float(y.double().norm())) <= 1e-12 * 8
    C = mat(cm(8, 8, torch.float32, 3, "cpu"))
    A, B = mat(x), mat(y)
    sl.gemm_bias_act(1.0, A, A, None, "identity", 0.0, None, C)
    A.storage = B.storage
    sl.gemm_bias_act(1.0, A, A, None, "identity", 0.0, None, C)
    y64 = y.double()
    within(C.to_dense(), y64 @ y64, 2.0 ** -24 * (12 * (y64.abs() @ y64.abs()) + (y64 @ y64).abs()))


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("dt", HALF)
def test_clip_types_share_memory(dev, dt):
    """16-bit matrices and float32 ones over the same memory: not 'in place', whatever their leading dimensions."""
    buf = torch.zeros(64, dtype=torch.float32, device=dev)
    half = buf.view(dt)
    x = half[:32].view(4, 8).t()                             # 8 x 4, at the front of the buffer
    x.copy_(torch.arange(1, 33, device=dev).view(4, 8).t())
    was = buf.clone()
    for y in (buf[:32].view(4, 8).t(), buf.as_strided((8, 4), (1, 16)), buf[8:40].view(4, 8).t()):
        for limit in (1e9, 1.0):
            with pytest.raises(SlateError, match="overlap"):
                sl.clip_norm(limit, [mat(x)], [mat(y)])
    a, b = half[:8][:, None], buf[:8][:, None]               # one column each
    with pytest.raises(SlateError, match="overlap"):
        sl.clip_norm(1.0, [mat(a)], [mat(b)])
    assert torch.equal(buf, was)
    y = buf[32:].view(4, 8).t()
    sl.clip_norm(1e9, [mat(x)], [mat(y)])
    assert torch.equal(y, x.float())


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("dt,out", CLIP_TYPES[:6])
@pytest.mark.parametrize("pad", [0, 3])
def test_clip_far_factors(dev, dt, out, pad):
    """Factors that the sums' type does not hold, or not with all its bits: the
    scaled elements are off as others are (4 w and the store's rounding; a
    subnormal result by its half step once more)."""
    rt = torch.float64 if dt == torch.float64 else torch.float32
    top = math.frexp(torch.finfo(dt).max)[1]
    step = torch.finfo(out).tiny * torch.finfo(out).eps
    for size in (2.0 ** (top - 7), 2.0 ** (top - 12)):
        unit = cm(60, 33, dt, 1, dev).double().clamp(-8, 8)
        x, y = cm(60, 33, dt, 1, dev, 1.0, pad), cm(60, 33, out, 2, dev, 1.0, pad)
        unit[3, 4], unit[5, 6] = 1 / size, 0.0
        norm = float(unit.norm())                                     # x = size unit, exactly
        for limit in (1.0, 1e-3, 1e-6, size * 2.0 ** -126, size * 2.0 ** -100, torch.finfo(rt).tiny, 1e-310, 5e-324):
            x.copy_(unit * size)
            part, e = math.frexp(limit)
            want = torch.ldexp(torch.ldexp(unit * (part / norm), torch.tensor(e // 2, device=dev)),
                               torch.tensor(e - e // 2, device=dev))
            s = float(sl.clip_norm(limit, [mat(x)], [mat(y)]))
            assert abs(s / size - norm) <= 2000 * 2.0 ** -53 * norm
            # the sum of 1980 squares, the product, the store; what ends subnormal by half a step of
            # either the product or the store
            rel = u_of(out) + 4 * w_of(out) + 2000 * 2.0 ** -53
            assert ((y.double() - want).abs() <= rel * want.abs() + step).all(), (size, limit)
            if dt == out:
                sl.clip_norm(limit, [mat(x)])
                assert torch.equal(x, y)


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("trans", [False, True])
def test_no_tokens_in_a_larger_buffer(dev, dt, trans):
    """The zero bias gradient of an empty batch does not reach what lies around the vector."""
    A, B = cm(16, 32, dt, 1, dev), torch.empty(0, 32, dtype=dt, device=dev).t()
    E = mat(torch.empty(16, 0, dtype=dt, device=dev).t(), True) if trans else mat(torch.empty(0, 16, dtype=dt, device=dev).t())
    whole = torch.ones(2, 24, dtype=dt, device=dev).t()
    b = sl.Matrix.fromScaLAPACK(16, 1, whole, nb=8)
    sl.gemm_bias_act_grad(1.0, mat(A), mat(B), "gelu", E, E, None, None, b)
    assert (whole[:16, 0] == 0).all() and (whole[16:] == 1).all() and (whole[:, 1] == 1).all()


class _Meddling:
    """A storage's tile table that another thread changes right after a call of `name`."""

    def __init__(self, table, name, act):
        self._table, self._name, self._act = table, name, act

    def __getattr__(self, k):
        f = getattr(self._table, k)
        if k != self._name:
            return f

        def call(*a):
            r = f(*a)
            act, self._act = self._act, None
            if act is not None:
                act()
            return r
        return call


def _two_sides():
    """An 8 x 8 matrix with a buffer on either side (both in host memory here)."""
    from slate_amd.core.storage import DEV, HOST
    x = cm(8, 8, torch.float64, 1, "cpu")
    s = mat(x, nb=4).storage
    y = s.allocate_local(DEV)
    s.prepare_local(DEV)
    return x, y, s, HOST, DEV


def test_change_while_a_side_is_made_valid(monkeypatch):
    """A tile modified on the other side after the scan of the states is copied by the next call."""
    from slate_amd.utils.debug import Debug
    x, y, s, HOST, DEV = _two_sides()
    todo = [True]

    def enabled():                                       # asked between the scan and its end
        if todo:
            todo.clear()
            x[0, 0] = 7.0
            s.tileModified(0, 0, HOST, True)
        return False

    monkeypatch.setattr(Debug, "enabled", enabled)
    s.tileModified(1, 1, HOST, True)
    s.prepare_local(DEV)
    s.prepare_local(DEV)
    assert not todo and y[0, 0] == 7.0 and torch.equal(x, y[:8, :8])


def test_change_while_a_side_is_marked():
    """A tile modified on the other side right after a mark is marked by the next one."""
    from slate_amd import _native
    x, y, s, HOST, DEV = _two_sides()
    s.table = _Meddling(s.table, "mark_all", lambda: s.tileModified(0, 0, HOST, True))
    s.mark_local_modified(DEV)
    assert s.table.state(0, 0, DEV) == _native._host.MOSI_Invalid
    s.mark_local_modified(DEV)
    assert s.table.state(0, 0, DEV) == _native._host.MOSI_Modified
    assert s.table.state(0, 0, HOST) == _native._host.MOSI_Invalid


def test_debug_checks_where_states_are_remembered(monkeypatch):
    """With the debug checks on, a call that remembers its operands runs them too."""
    from slate_amd import _native
    from slate_amd.utils.debug import Debug
    monkeypatch.setattr(Debug, "_on", False)
    x, y, s, HOST, DEV = _two_sides()
    A = mat(x, nb=4)
    A.storage = s
    sl.global_norm([A])
    x[1, 2] += 1.0                                       # both sides are valid, and differ now
    sl.global_norm([A])
    C = mat(cm(8, 8, torch.float64, 2, "cpu"))
    monkeypatch.setattr(Debug, "_on", True)
    for call in (lambda: s.prepare_local(HOST), lambda: s.prepare_local(DEV), lambda: sl.global_norm([A]),
                 lambda: sl.clip_norm(1.0, [A]),
                 lambda: sl.gemm_bias_act(1.0, A, A, None, "relu", 0.0, None, C)):
        with pytest.raises(SlateError, match="MOSI"):
            call()
    monkeypatch.setattr(Debug, "_on", False)
    s = mat(x, nb=4).storage
    s.table.set_state(0, 0, HOST, _native._host.MOSI_Shared | _native._host.MOSI_OnHold)
    s.mark_local_modified(HOST)
    monkeypatch.setattr(Debug, "_on", True)
    with pytest.raises(SlateError, match="MOSI"):
        s.mark_local_modified(HOST)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("k", [3, 641, 4096, 4099])
@pytest.mark.parametrize("pad,off", [(0, 0), (3, 1), (5, 0)])
def test_few_columns(dt, k, pad, off):
    """Up to 16 columns and both operands along k, 1024 rows or more: whole batches of slabs and a
    ragged end of K, columns and rows past the matrix, operands off 16 bytes."""
    for m, n in ((1024, 1), (1030, 2), (4096, 7), (1024, 15), (1030, 16)):
        Product(dt, "cuda", m, n, k, "T", "N", act="gelu", bias=1 + n % 2, pad=pad, off=off, cpad=pad).check()
        Gated(dt, "cuda", m, n, k, "T", "N", pad=pad, off=off).check()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("m,n,k", [(5120, 15, 5888), (5120, 8, 5888), (4096, 15, 5888), (8192, 16, 5888), (5121, 9, 5887),
                                   (4097, 16, 1000), (1023, 16, 5888), (1024, 17, 5888)])
def test_few_columns_borders(dt, m, n, k):
    """Either side of the rules that send few columns to tiles with K in pieces."""
    Product(dt, "cuda", m, n, k, "T", "N", act="silu").check()
    Gated(dt, "cuda", m, n, k, "T", "N").check()


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("count", [71, 72, 73, 143, 144, 145])
@pytest.mark.parametrize("empty", [0, 3])
def test_clip_launches(dev, count, empty):
    """Matrices that fill one launch or two of 72 exactly, and one less and more; empty ones take no place."""
    xs = clip_case(torch.float32, dev, [(1 + 7 * i % 23, 1 + i % 11) for i in range(count)], 1.0)
    s, f = clip_want(xs, 2.0)
    no = clip_case(torch.float32, dev, [(0, 4), (5, 0), (0, 0)][:empty])
    a = [mat(x) for x in no[:1] + xs[:50] + no[1:] + xs[50:]]
    ys = [torch.full_like(x, float("nan")) for x in xs]
    b = [mat(y) for y in no[:1] + ys[:50] + no[1:] + ys[50:]]
    for got in (sl.clip_norm(2.0, a, b), sl.clip_norm(2.0, a)):
        # the squares of 24 bits are exact in 53, their sum of n terms is off by n halves of an ulp
        n = sum(x.numel() for x in xs)
        assert abs(float(got) - s) <= (n + 4) * 2.0 ** -53 * s
    for x, y, was in zip(xs, ys, clip_case(torch.float32, dev, [(1 + 7 * i % 23, 1 + i % 11) for i in range(count)], 1.0)):
        want = was.double() * f
        assert ((y.double() - want).abs() <= 4 * 2.0 ** -24 * want.abs()).all()
        assert torch.equal(x, y)


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("src", TYPES)
@pytest.mark.parametrize("dst", TYPES)
@pytest.mark.parametrize("uplo", ["L", "U"])
@pytest.mark.parametrize("trans", ["N", "T"])
def test_copy_half_triangle(dev, src, dst, uplo, trans):
    """One triangle's copy to and from the 16-bit types; the other keeps its elements."""
    if src not in HALF and dst not in HALF:
        pytest.skip("the other kernels")
    for m, n in ((67, 45), (300, 33), (33, 300), (1, 5), (5, 1)):
        x = cm(*((m, n) if trans == "N" else (n, m)), src, 3, dev)
        y = cm(m, n, dst, 4, dev, 1.0, 3)
        keep = y.clone()
        ops.gecopy(x, y, uplo, trans)
        want = (x if trans == "N" else x.t()).cpu().to(dst)
        tri = torch.ones(m, n).tril().bool() if uplo == "L" else torch.ones(m, n).triu().bool()
        assert torch.equal(y.cpu(), torch.where(tri, want, keep.cpu()))


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("src,dst", [(torch.float32, torch.bfloat16), (torch.float16, torch.float64), (torch.bfloat16,) * 2])
def test_copy_half_kinds(dev, src, dst):
    """sl.copy of triangular and Hermitian matrices to and from the 16-bit types."""
    for uplo in (sl.Uplo.Lower, sl.Uplo.Upper):
        for kind in (sl.TriangularMatrix, sl.HermitianMatrix):
            x, y = cm(45, 45, src, 3, dev), cm(45, 45, dst, 4, dev)
            keep = y.clone()
            sl.copy(kind(uplo, mat(x, nb=16)), kind(uplo, mat(y, nb=16)))
            tri = torch.ones(45, 45).tril().bool()
            tri = tri if uplo == sl.Uplo.Lower else tri.t()
            assert torch.equal(y.cpu(), torch.where(tri, x.cpu().to(dst), keep.cpu()))


def precise_grads(dt, dev, m, n, k, ta="T", tb="N", act="gelu", pad=0, off=0, gated=False, opts={"PreciseGradient": True},
                  which=("A1", "A2", "B")):
    """Gradients with what the rounding of dZ leaves over, and [(got, wanted, bound)].

    Two parts of 16 bits hold dZ to u^2 of itself and half the smallest step; the
    products' sums have twice the terms."""
    u, w = u_of(dt), w_of(dt)
    g = Gated(dt, dev, m, n, k, ta, tb, act, pad, off)
    a1, a2, b = g.dense()
    z1, z2, c = g.Z1.double(), g.Z2.double(), g.G.double()
    v, s = act64(act, z1)
    left = (u * u if u > w else 0) + 4 * w
    d = {x: cm(*getattr(g, x).shape, dt, 9, dev) if x in which else None for x in ("A1", "A2", "B")}
    t = {"A1": ta == "T", "A2": ta == "T", "B": tb == "T"}
    out = [None if d[x] is None else mat(d[x], t[x]) for x in ("A1", "A2", "B")]
    A1, A2, B = g.handles()
    bt, a1t, a2t = b.t().contiguous(), a1.t().contiguous(), a2.t().contiguous()
    one = c * z2 if gated else c
    dz1, f1 = one * s, 32 * w * (1 + z1.abs()) * one.abs() + left * (one * s).abs() + tiny(dt)
    terms = [("A1", dz1 @ bt, f1 @ bt.abs() + 2 * (n + 4) * w * (dz1.abs() @ bt.abs()))]
    bsum, bbound = a1t @ dz1, a1t.abs() @ f1 + 4 * (m + 4) * w * (a1t.abs() @ dz1.abs())
    if gated:
        sl.gemm_gated_grad(A1, A2, B, act, mat(g.Z1), mat(g.Z2), mat(g.G), *out, opts)
        dz2, f2 = c * v, 32 * w * (1 + z1.abs()) * (c * z1).abs() + left * (c * v).abs() + tiny(dt)
        terms.append(("A2", dz2 @ bt, f2 @ bt.abs() + 2 * (n + 4) * w * (dz2.abs() @ bt.abs())))
        bsum, bbound = bsum + a2t @ dz2, bbound + a2t.abs() @ f2 + 4 * (m + 4) * w * (a2t.abs() @ dz2.abs())
    else:
        sl.gemm_bias_act_grad(1.0, A1, B, act, mat(g.Z1), mat(g.G), out[0], out[2], None, opts)
    terms.append(("B", bsum, bbound))
    return [(d[x].t() if t[x] else d[x], want, e + tiny(dt) + u * (want.abs() + e)) for x, want, e in terms if x in which]


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("ta,tb", ["TN", "NN", "NT", "TT"])
@pytest.mark.parametrize("gated", [False, True])
def test_precise_gradient(dev, dt, ta, tb, gated):
    for m, n, k, act, pad, off in ((70, 33, 50, "gelu", 0, 0), (48, 1, 40, "silu", 8, 0), (131, 67, 75, "gelu_tanh", 3, 1),
                                   (1, 1, 1, "relu", 0, 0)):
        for which in (("A1", "A2", "B"), ("B",), ("A1", "B")):
            for got, want, e in precise_grads(dt, dev, m, n, k, ta, tb, act, pad, off, gated, which=which):
                within(got, want, e)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", HALF)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m,n,k,pad", [(1024, 2048, 512, 0), (4000, 3, 640, 0), (600, 5000, 128, 0), (2051, 2049, 2053, 1),
                                       (328, 264, 200, 0), (2560, 515, 1024, 0)])
def test_precise_gradient_sizes(dt, gated, m, n, k, pad):
    """K in pieces that begin in any of two or four products, short last steps, operands laid out anew."""
    first = precise_grads(dt, "cuda", m, n, k, pad=pad, gated=gated)
    for got, want, e in first:
        within(got, want, e)
    for (x, _, _), (y, _, _) in zip(first, precise_grads(dt, "cuda", m, n, k, pad=pad, gated=gated)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("dt", HALF)
def test_precise_gradient_choice(dev, dt):
    """The option lowers the error of dA and dB, changes nothing of 32 bits, and keeps infinities."""
    err = {}
    for on in (False, True):
        got = precise_grads(dt, dev, 96, 64, 80, opts={sl.Option.PreciseGradient: on}, gated=True)
        err[on] = [float((x.double() - w).norm() / w.norm()) for x, w, _ in got]
    # one rounding of random relative size against two of the same: by 2^0.5, a tenth less for chance
    assert all(a > 1.27 * b for a, b in zip(err[False], err[True])), err
    a, b = (precise_grads(torch.float32, dev, 40, 24, 32, opts=o) for o in (None, {"PreciseGradient": True}))
    assert all(torch.equal(x[0], y[0]) for x, y in zip(a, b))
    one = torch.ones(1, 1, dtype=dt, device=dev)
    big = torch.full((1, 1), torch.finfo(dt).max, dtype=dt, device=dev)
    for z2, g, want in ((big, big, float("inf")), (big, one, float(big)), (one * float("nan"), one, float("nan"))):
        d = torch.empty(1, 1, dtype=dt, device=dev)
        sl.gemm_gated_grad(mat(one), mat(one), mat(one), "identity", mat(one), mat(z2), mat(g), mat(d), None, None,
                           {"PreciseGradient": True})
        assert float(d) == want or want != want and d.isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("gated", [False, True])
def test_precise_gradient_graph(gated):
    """The option's backward pass captured and replayed, with eager work between."""
    s, _ = block(torch.bfloat16, "cuda", 77, 256, 520)
    H = {n: mat(v, n in ("wg", "wu", "dwg", "dwu")) for n, v in s.items()}
    for n in ("z1", "z2", "dh"):
        s[n].copy_(cm(*s[n].shape, torch.bfloat16, 30 + len(n), "cuda"))
    names = ("dwg", "dwu", "dx") if gated else ("dwg", "dx")
    opts = {"PreciseGradient": True}

    def step():
        if gated:
            sl.gemm_gated_grad(H["wg"], H["wu"], H["x"], "silu", H["z1"], H["z2"], H["dh"], H["dwg"], H["dwu"], H["dx"], opts)
        else:
            sl.gemm_bias_act_grad(1.0, H["wg"], H["x"], "silu", H["z1"], H["dh"], H["dwg"], H["dx"], None, opts)

    step()
    want = {n: s[n].clone() for n in names}
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for _ in range(3):
        for n in names:
            s[n].fill_(float("nan"))
        g.replay()
        torch.cuda.synchronize()
        for n in names:
            assert torch.equal(s[n], want[n]), n
        step()
        torch.cuda.synchronize()

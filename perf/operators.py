"""The fused products of a feed-forward block and the clipping of its gradients: inputs, calls, plain forms, exact values.

Tensors are held as a training or serving program holds them: tokens (and the rows of a weight) one after the
other, which is the column-major layout of the library's matrices.  X of t tokens with k features is a t x k
tensor, that is the k x t matrix; a weight stored as m x k (``stored`` "T") is the k x m matrix whose transposed
view enters the product, one stored as k x m ("N") enters as it is.  ``pad`` is what a leading dimension has
beyond the row: 0 and multiples of 8 keep every row on 16 bytes, odd ones do not.
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "f64": torch.float64}
_ACTS = ("identity", "relu", "gelu", "gelu_tanh", "silu")


# ------------------------------------------------------------------ cases
def _product(name, dt, t, k, m, act, bias=True, res=False, keep=False, stored="T", pad=0):
    return dict(name=name, op="product", dt=dt, t=t, k=k, m=m, act=act, bias=bias, res=res, keep=keep,
                stored=stored, pad=pad)


def _grad(name, dt, t, k, m, act, bias=True, stored="T", pad=0):
    return dict(name=name, op="product_grad", dt=dt, t=t, k=k, m=m, act=act, bias=bias, stored=stored, pad=pad)


def _gated(name, dt, t, k, m, act, keep=False, stored="T", pad=0):
    return dict(name=name, op="gated", dt=dt, t=t, k=k, m=m, act=act, keep=keep, stored=stored, pad=pad)


def _gated_grad(name, dt, t, k, m, act, stored="T", pad=0):
    return dict(name=name, op="gated_grad", dt=dt, t=t, k=k, m=m, act=act, stored=stored, pad=pad)


def _clip(name, dt, out, blocks, d, f, vectors, limit):
    return dict(name=name, op="clip", dt=dt, out=out, blocks=blocks, d=d, f=f, vectors=vectors, limit=limit)


def listed():
    return [
        # one token through a projection: serving's latency, bound by reading the weight once
        _product("product 1 token", "bf16", 1, 4096, 4096, "gelu"),
        # a ragged batch of requests through the projection back, onto the residual stream
        _product("product 33 tokens residual", "f16", 33, 8192, 2048, "identity", res=True),
        # a training step's widest projection, the pre-activation kept for the backward pass
        _product("product training", "bf16", 8192, 4096, 16384, "gelu_tanh", keep=True),
        # single precision, an odd number of tokens, a weight stored the other way round
        _product("product single precision", "f32", 1001, 1024, 4096, "silu", res=True, stored="N"),
        # backward of a training projection: both gradients and the bias gradient
        _grad("product grad training", "bf16", 4096, 4096, 8192, "gelu"),
        # the same at odd sizes, where no row lies on 16 bytes
        _grad("product grad odd", "f32", 777, 1001, 1503, "relu"),
        # one token through the gated block: two weights to read
        _gated("gated 1 token", "f16", 1, 4096, 8192, "silu"),
        # a gated block over a long batch, both projections kept for the backward pass
        _gated("gated training", "bf16", 8192, 4096, 8192, "silu", keep=True),
        # its backward pass: three gradients
        _gated_grad("gated grad training", "bf16", 4096, 4096, 8192, "silu"),
        # a small model's, in half precision over a ragged batch
        _gated_grad("gated grad ragged", "f16", 515, 1024, 2560, "gelu"),
        # the gradients of a small model: many small matrices and vectors, where launches count
        _clip("clip small", "f32", "f32", 6, 256, 1024, 4, 1.0),
        # a large one's, 16-bit gradients into single precision for the optimizer
        _clip("clip large", "bf16", "f32", 4, 4096, 16384, 4, 1.0),
    ]


def _span(rng, lo, hi, even=0.5):
    """A size spread over its logarithm; half of them whole multiples of 64 (where they are that large)."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(lo, v // 64 * 64) if v >= 64 and rng.random() < even else v


def draw(rng):
    op = rng.choice(("product", "product", "product_grad", "gated", "gated_grad", "clip"))
    dt = rng.choice(("bf16", "bf16", "bf16", "f16", "f16", "f32", "f32", "f64"))
    if op == "clip":
        out = dt if dt in ("f32", "f64") or rng.random() < 0.5 else "f32"
        d = _span(rng, 16, 2048)
        vectors = rng.randint(0, 8)
        return dict(op=op, dt=dt, out=out, blocks=rng.randint(1, 60 // (6 + vectors)), d=d, f=_span(rng, d, 4 * d),
                    vectors=vectors, limit=rng.choice((0.5, 1.0, 1e9)))
    k, m = _span(rng, 16, 8192), _span(rng, 16, 8192)
    t = _span(rng, 1, 8192, 0.25)
    per = {"product": 2, "product_grad": 4, "gated": 4, "gated_grad": 8}[op] * k * m
    t = max(1, min(t, int(8e11 // per)))
    c = dict(op=op, dt=dt, t=t, k=k, m=m, act=rng.choice(_ACTS), stored=rng.choice("TTN"),
             pad=rng.choice((0, 0, 0, 8, 24, 5)))
    if op == "product":
        c.update(bias=rng.random() < 0.7, res=rng.random() < 0.5, keep=rng.random() < 0.4)
    elif op == "product_grad":
        c.update(bias=rng.random() < 0.7)
    elif op == "gated":
        c.update(keep=rng.random() < 0.4)
    return c


# ----------------------------------------------------------------- inputs
def _shapes(c):
    """The gradients of a model: for each block four d x d matrices, two d x f ones, and vectors."""
    d, f = c["d"], c["f"]
    return ([(d, d)] * 4 + [(f, d), (d, f)] + [(1, d)] * c["vectors"]) * c["blocks"]


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = _TYPES[c["dt"]]

    def rows(n, w, std, pad=0):
        x = torch.empty(n, w + pad, dtype=dt, device="cuda")
        return x.normal_(0.0, std, generator=g)[:, :w]

    s = {"case": c}
    if c["op"] == "clip":
        s["x"] = [rows(a, b, 0.02) for a, b in _shapes(c)]
        s["y"] = [torch.empty(a, b, dtype=_TYPES[c["out"]], device="cuda") for a, b in _shapes(c)]
    else:
        t, k, m, pad = c["t"], c["k"], c["m"], c["pad"]
        weight = (m, k) if c["stored"] == "T" else (k, m)
        s["x"] = rows(t, k, 1.0, pad)
        s["w"] = rows(*weight, k ** -0.5, pad)
        gated = c["op"].startswith("gated")
        if gated:
            s["w2"] = rows(*weight, k ** -0.5, pad)
        if c["op"].endswith("grad"):
            s["dc"] = rows(t, m, 0.1)
            s["z"] = rows(t, m, 1.0)
            s["dx"], s["dw"] = torch.empty(t, k, dtype=dt, device="cuda"), torch.empty(weight, dtype=dt, device="cuda")
            if gated:
                s["z2"] = rows(t, m, 1.0)
                s["dw2"] = torch.empty_like(s["dw"])
            elif c["bias"]:
                s["db"] = torch.empty(m, dtype=dt, device="cuda")
        else:
            s["c"] = torch.empty(t, m, dtype=dt, device="cuda")
            if c["keep"]:
                s["z"] = torch.empty_like(s["c"])
                if gated:
                    s["z2"] = torch.empty_like(s["c"])
            if not gated:
                s["b"] = rows(1, m, 0.5)[0] if c["bias"] else None
                s["r"] = rows(t, m, 1.0) if c["res"] else None
    if own:
        s["h"] = _handles(s)
    return s


def _handles(s):
    """The library's matrices over the same memory, which a program makes once."""
    import slate_amd as sl

    def matrix(x):
        if isinstance(x, list):
            return [matrix(y) for y in x]
        x = x.t() if x.dim() == 2 else x[:, None]
        return sl.Matrix.fromLAPACK(x.shape[0], x.shape[1], x, nb=1024)

    h = {n: matrix(x) for n, x in s.items() if n != "case" and x is not None}
    if s["case"].get("stored") == "T":
        h.update({n: h[n].transpose() for n in ("w", "w2", "dw", "dw2") if n in h})
    return h


# ------------------------------------------------------------------- plain
def _wide(x):
    return x if x.dtype == torch.float64 else x.float()


def _act(name, z):
    if name == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    if name == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _slope(name, z):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        h = torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + h) + 0.5 * z * (1 - h * h) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z)
    if name == "silu":
        e = 1 / (1 + torch.exp(-z))
        return e * (1 + z * (1 - e))
    return torch.ones_like(z)


def _weight(c, w):
    """The m x k matrix of a weight, however it is stored."""
    return _wide(w if c["stored"] == "T" else w.t())


def _as_stored(c, g):
    return g if c["stored"] == "T" else g.t().contiguous()


def _plain(s):
    c = s["case"]
    if c["op"] == "clip":
        norm = torch.sqrt(sum((x.double() * x.double()).sum() for x in s["x"]))
        part = torch.clamp(c["limit"] / norm, max=1.0)
        return {"norm": norm, "y": [(_wide(x) * part.to(_wide(x).dtype)).to(_TYPES[c["out"]]) for x in s["x"]]}
    dt, x, w = s["x"].dtype, _wide(s["x"]), _weight(c, s["w"])
    if c["op"] == "product":
        z = x @ w.t()
        if c["bias"]:
            z = z + _wide(s["b"])
        y = _act(c["act"], z)
        if c["res"]:
            y = y + _wide(s["r"])
        return {"c": y.to(dt), **({"z": z.to(dt)} if c["keep"] else {})}
    if c["op"] == "gated":
        z, z2 = x @ w.t(), x @ _weight(c, s["w2"]).t()
        y = _act(c["act"], z) * z2
        return {"c": y.to(dt), **({"z": z.to(dt), "z2": z2.to(dt)} if c["keep"] else {})}
    z, dc = _wide(s["z"]), _wide(s["dc"])
    if c["op"] == "product_grad":
        dz = dc * _slope(c["act"], z)
        out = {"dx": (dz @ w).to(dt), "dw": _as_stored(c, (dz.t() @ x).to(dt))}
        return {**out, "db": dz.sum(0).to(dt)} if c["bias"] else out
    dz, dz2 = dc * _wide(s["z2"]) * _slope(c["act"], z), dc * _act(c["act"], z)
    return {"dx": (dz @ w + dz2 @ _weight(c, s["w2"])).to(dt), "dw": _as_stored(c, (dz.t() @ x).to(dt)),
            "dw2": _as_stored(c, (dz2.t() @ x).to(dt))}


# --------------------------------------------------------------------- run
def run(state):
    if not own:
        return _plain(state)
    import slate_amd as sl
    s, c, h = state, state["case"], state["h"]
    if c["op"] == "clip":
        return {"norm": sl.clip_norm(c["limit"], h["x"], h["y"]), "y": s["y"]}
    if c["op"] == "product":
        sl.gemm_bias_act(1.0, h["w"], h["x"], h.get("b"), c["act"], 1.0, h.get("r"), h["c"], h.get("z"))
        return {n: s[n] for n in ("c", "z") if n in s}
    if c["op"] == "gated":
        sl.gemm_gated(h["w"], h["w2"], h["x"], c["act"], h["c"], h.get("z"), h.get("z2"))
        return {n: s[n] for n in ("c", "z", "z2") if n in s}
    if c["op"] == "product_grad":
        sl.gemm_bias_act_grad(1.0, h["w"], h["x"], c["act"], h["z"], h["dc"], h["dw"], h["dx"], h.get("db"))
        return {n: s[n] for n in ("dx", "dw", "db") if n in s}
    sl.gemm_gated_grad(h["w"], h["w2"], h["x"], c["act"], h["z"], h["z2"], h["dc"], h["dw"], h["dw2"], h["dx"])
    return {n: s[n] for n in ("dx", "dw", "dw2")}


# -------------------------------------------------------------------- work
def work(case):
    c = case
    e = {"bf16": 2, "f16": 2, "f32": 4, "f64": 8}
    if c["op"] == "clip":
        n = sum(a * b for a, b in _shapes(c))
        return {"bytes": n * (e[c["dt"]] + e[c["out"]]) + 8, "flops": 3 * n}
    t, k, m = c["t"], c["k"], c["m"]
    if c["op"] == "product":
        words = m * k + k * t + m * t * (1 + c["res"] + c["keep"]) + m * c["bias"]
        flops = 2 * m * k * t
    elif c["op"] == "gated":
        words, flops = 2 * m * k + k * t + m * t * (1 + 2 * c["keep"]), 4 * m * k * t
    elif c["op"] == "product_grad":
        words, flops = 2 * m * k + 2 * k * t + 2 * m * t + m * c["bias"], 4 * m * k * t
    else:
        words, flops = 4 * m * k + 2 * k * t + 3 * m * t, 8 * m * k * t
    return {"bytes": words * e[c["dt"]], "flops": flops}


# ------------------------------------------------------------------- exact
def _erf_cdf(z):
    """The normal distribution's function."""
    return 0.5 * torch.special.erfc(-z / 2 ** 0.5)


def _exact_act(name, z):
    """(value, derivative) of the activation in 64 bits, by its definition."""
    one = torch.ones_like(z)
    if name == "relu":
        return z.clamp(min=0.0), (z > 0).double()
    if name == "gelu":
        p = _erf_cdf(z)
        return z * p, p + z * torch.exp(-z.square() / 2) / (2 * math.pi) ** 0.5
    if name == "gelu_tanh":
        u = (2 / math.pi) ** 0.5 * (z + 0.044715 * z ** 3)
        p = torch.sigmoid(2 * u)              # (1 + tanh u) / 2
        return z * p, p + z * p * (1 - p) * 2 * (2 / math.pi) ** 0.5 * (1 + 0.134145 * z ** 2)
    if name == "silu":
        p = torch.sigmoid(z)
        return z * p, p + z * p * (1 - p)
    return z, one


def exact(case, seed):
    c = case
    s = prepare(c, seed)
    if c["op"] == "clip":
        norm = math.sqrt(math.fsum(float(torch.linalg.vector_norm(x.double())) ** 2 for x in s["x"]))
        return {"norm": torch.tensor(norm, dtype=torch.float64),
                "y": [x.double() * min(1.0, c["limit"] / norm) for x in s["x"]]}
    x, w = s["x"].double(), s["w"].double()
    w = w.mT if c["stored"] == "N" else w
    back = (lambda g: g) if c["stored"] == "T" else (lambda g: g.mT.contiguous())
    if c["op"] == "product":
        z = torch.matmul(x, w.mT)
        z = z + s["b"].double() if c["bias"] else z
        y = _exact_act(c["act"], z)[0]
        y = y + s["r"].double() if c["res"] else y
        return {"c": y, **({"z": z} if c["keep"] else {})}
    w2 = None
    if "w2" in s:
        w2 = s["w2"].double()
        w2 = w2.mT if c["stored"] == "N" else w2
    if c["op"] == "gated":
        z, z2 = torch.matmul(x, w.mT), torch.matmul(x, w2.mT)
        return {"c": z2 * _exact_act(c["act"], z)[0], **({"z": z, "z2": z2} if c["keep"] else {})}
    value, slope = _exact_act(c["act"], s["z"].double())
    dc = s["dc"].double()
    if c["op"] == "product_grad":
        dz = slope * dc
        out = {"dx": torch.matmul(dz, w), "dw": back(torch.matmul(dz.mT, x))}
        return {**out, "db": torch.matmul(dz.new_ones(1, dz.shape[0]), dz)[0]} if c["bias"] else out
    dz, dz2 = slope * s["z2"].double() * dc, value * dc
    return {"dx": torch.matmul(dz2, w2) + torch.matmul(dz, w), "dw": back(torch.matmul(dz.mT, x)),
            "dw2": back(torch.matmul(dz2.mT, x))}

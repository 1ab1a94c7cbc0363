"""Fused products of a feed-forward block, their gradients, and the clipping
of many gradients by their common norm.

* :func:`gemm_bias_act`  C = act(alpha op(A) op(B) + bias) + beta R
* :func:`gemm_gated`     C = act(op(A1) op(B)) o (op(A2) op(B))
* their backward passes :func:`gemm_bias_act_grad`, :func:`gemm_gated_grad`
* :func:`clip_norm`      B_i = min(1, max_norm / |A|) A_i over a list of matrices,
  :func:`global_norm` the norm alone

They stand next to ``gemm``, ``norm`` and ``scale``: the same matrices, views,
grids and streams.  Element types are bfloat16, float16, float32 and float64
(``clip_norm`` takes complex matrices too); a call's matrices share one type.
Sums, biases, activations and norms are computed in 32 bits (64 for float64)
and rounded once, to nearest even, when an output is stored.

MI355X design: one MFMA launch per product with the epilogue on the
accumulators (csrc/hip/gemm_act.hpp); a gated product keeps both projections
of a tile in one workgroup, so neither is written unless asked for; the
backward pass is one elementwise pass (csrc/hip/act_grad.hip) and one launch
per operand gradient.  On p x q ranks every rank gathers its rows of op(A)
and its columns of op(B) (one broadcast per tile column and row, as SUMMA
moves them) and makes its block of C with one launch: the epilogue needs the
whole sum, and partial sums in 16 bits would be rounded on the way.

Calls enqueue on the current stream of the matrices' device, never
synchronise, and can be captured into a hipGraph (on one rank).
"""
from __future__ import annotations

import torch

from .. import ops
from .._native import REAL_CODE, kmod, raw_stream
from ..core.enums import Activation, Op
from ..core.exceptions import SlateError
from ..core.storage import DEV
from ..utils.trace import trace_block
from ._panels import col_bcast, row_bcast
from ._util import grid_of, tiles_local_before
from .blas3 import _copy_in, _copy_out, _fresh, _single

PLAIN, GATED, SUM, PAIR = 0, 1, 2, 3
_ACT = {a: i for i, a in enumerate(Activation)}
_ACT.update({a.name.lower(): i for a, i in list(_ACT.items())})
_BYTES = {torch.bfloat16: 2, torch.float16: 2, torch.float32: 4, torch.float64: 8}


# ------------------------------------------------------------------ operands
class _Opd:
    """One rank's strided column-major operand: address, leading dimension,
    stored shape, whether it enters transposed, and the tensor that owns it."""

    __slots__ = ("ptr", "ld", "rows", "cols", "trans", "t")

    def __init__(self, ptr, ld, rows, cols, trans, t):
        self.ptr, self.ld, self.rows, self.cols, self.trans, self.t = ptr, ld, rows, cols, trans, t

    @property
    def T(self):
        return _Opd(self.ptr, self.ld, self.rows, self.cols, not self.trans, self.t)

    @property
    def op(self):
        return 'T' if self.trans else 'N'

    @property
    def m(self):
        return self.cols if self.trans else self.rows

    @property
    def n(self):
        return self.rows if self.trans else self.cols


_NONE = _Opd(0, 0, 0, 0, False, None)


def _of_tensor(t, rows, cols, trans=False, name="matrix"):
    ld = t.stride(1) if cols > 1 else -(-max(rows, 1) // 8) * 8
    if cols > 1 and ld < rows:
        raise SlateError(f"{name}: columns overlap (leading dimension {ld} < {rows} rows)")
    return _Opd(t.data_ptr(), ld, rows, cols, trans, t)


def _opd(M, name="matrix"):
    """The (one) rank's operand of a view."""
    s = M.storage
    if M._mt == s.mt and M._nt == s.nt and not (M.ioffset or M.joffset or M.row0_offset or M.col0_offset) \
            and M.last_mb is None and M.last_nb is None and s.origin_slot is not None:
        t, rows, cols = s.prepare_local(s.origin_slot), s.bc.mloc, s.bc.nloc
    else:
        t = M.local_block().data
        rows, cols = t.shape
    return _of_tensor(t, rows, cols, M._op != Op.NoTrans, name)


def _t(M):
    """Transposed view (the element types are real: ConjTrans is Trans)."""
    return None if M is None else M._clone(_op=Op.NoTrans if M._op != Op.NoTrans else Op.Trans)


def _span(x):
    return x.ptr, x.ptr + ((x.cols - 1) * x.ld + x.rows) * _BYTES[x.t.dtype] if x.rows and x.cols else x.ptr


def _overlap(x, y):
    """Do two operands share elements?  Blocks of one leading dimension are
    compared as rectangles, others by their address ranges."""
    (a0, a1), (b0, b1) = _span(x), _span(y)
    if a1 <= b0 or b1 <= a0:
        return False
    es = _BYTES[x.t.dtype]
    if y.t.dtype != x.t.dtype or (b0 - a0) % es or (x.cols > 1 and y.cols > 1 and x.ld != y.ld):
        return True
    ld = x.ld if x.cols > 1 else y.ld
    if x.rows > ld or y.rows > ld:
        return True
    dc, dr = divmod((b0 - a0) // es, ld)
    for c, r in ((dc, dr), (dc + 1, dr - ld)):
        if r < x.rows and -r < y.rows and c < x.cols and -c < y.cols:
            return True
    return False


def _outputs(outs, ins, names, in_names, same=()):
    """Outputs share no element with each other or with inputs; ``same`` lists
    (output, input) pairs that may be the same view (read, then written, by the
    same thread)."""
    for i, x in enumerate(outs):
        if x.t is None:
            continue
        for j, y in enumerate(ins):
            if y.t is None or ((i, j) in same and (x.ptr, x.ld, x.trans, x.t.dtype) == (y.ptr, y.ld, y.trans, y.t.dtype)):
                continue
            if _overlap(x, y):
                raise SlateError(f"output {names[i]} overlaps {in_names[j]}")
        for j in range(i):
            if outs[j].t is not None and _overlap(x, outs[j]):
                raise SlateError(f"outputs {names[i]} and {names[j]} overlap")


def _act(act):
    i = _ACT.get(act)
    if i is None:
        try:
            return _ACT[Activation.from_string(act)]
        except (KeyError, ValueError):
            raise SlateError(f"unknown activation {act!r}") from None
    return i


def _where(s):
    """Device of a storage's local buffer."""
    return s.local[s.origin_slot].device


def _check(mats, shapes, what):
    """Types, kinds, devices and shapes of a call's matrices ({name: M or None})."""
    first = None
    for name, M in mats.items():
        if M is None:
            continue
        s = M.storage
        if getattr(M, "_kind", "general") != "general" or s.bc is None:
            raise SlateError(f"{what}: {name} must be a general block-cyclic matrix")
        if first is None:
            first = s
            if s.dtype not in REAL_CODE:
                raise SlateError(f"{what}: element type {s.dtype} (bfloat16, float16, float32 or float64 are wanted)")
        elif s.dtype != first.dtype:
            raise SlateError(f"{what}: {name} has type {s.dtype}, the others {first.dtype}")
        if s.origin_slot is None:
            raise SlateError(f"{what}: {name} has no tiles (insertLocalTiles)")
        if _where(s) != _where(first):
            raise SlateError(f"{what}: {name} is on {_where(s)}, the others on {_where(first)}")
        m, n = shapes[name]
        if M.m() != m or M.n() != n:
            raise SlateError(f"{what}: {name} is {M.m()} x {M.n()}, {m} x {n} is wanted")
    return first


def _bias_shape(bias, m, n, what):
    """(shape to check, mode): one value per row (m x 1) or per column (1 x n)."""
    if bias is None:
        return (m, 1), 0
    if bias.n() == 1 and bias.m() == m:
        return (m, 1), 1
    if bias.m() == 1 and bias.n() == n:
        return (1, n), 2
    raise SlateError(f"{what}: bias is {bias.m()} x {bias.n()}, {m} x 1 or 1 x {n} is wanted")


def _inc(b):
    """Distance of a vector operand's elements."""
    return 1 if b.rows > 1 or b.cols <= 1 else b.ld


class _on:
    """The operands' device made current (launches and workspaces go there)."""

    def __init__(self, t):
        self.ctx = None
        if t.is_cuda and t.device.index != torch.cuda.current_device():
            self.ctx = torch.cuda.device(t.device)

    def __enter__(self):
        if self.ctx is not None:
            self.ctx.__enter__()

    def __exit__(self, *e):
        if self.ctx is not None:
            self.ctx.__exit__(*e)


def _launch(mode, alpha, A, B, C, bias=_NONE, bias_mode=0, act=0, beta=0.0, R=_NONE, Z=()):
    """One rank's product(s): operands as lists of _Opd, C not transposed."""
    t = C[0].t
    m, n, k = C[0].rows, C[0].cols, A[0].n
    if m == 0 or n == 0:
        return
    if alpha == 0:
        k = 0                                   # op(A) op(B) is not read
    if beta == 0:
        R = _NONE
    A, B, C = (list(x) + [_NONE] * (2 - len(x)) for x in (A, B, C))
    Z = [z or _NONE for z in Z] + [_NONE] * (2 - len(Z))
    if ops._FLOPS is not None:
        ops._FLOPS[0] += 2 * m * n * k * (1 if mode == PLAIN else 2)
    mod = kmod(t)
    nbytes = mod.gemm_act_ws(_BYTES[t.dtype], mode, m, n, k)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=t.device) if nbytes else None
    mod.gemm_act(REAL_CODE[t.dtype], mode, A[0].op, B[0].op, m, n, k, float(alpha),
                 A[0].ptr, A[0].ld, A[1].ptr, A[1].ld, B[0].ptr, B[0].ld, B[1].ptr, B[1].ld,
                 C[0].ptr, C[0].ld, C[1].ptr, C[1].ld, bias.ptr, _inc(bias), bias_mode, act, float(beta),
                 R.ptr, R.ld, Z[0].ptr, Z[0].ld, Z[1].ptr, Z[1].ld,
                 0 if ws is None else ws.data_ptr(), raw_stream(t))


def _like(x, rows, cols, trans=False):
    """Workspace beside operand x, columns on 16-byte (long ones on 128-byte) borders."""
    ld = -(-rows // 64) * 64 if rows >= 64 else -(-max(rows, 1) // 8) * 8
    t = torch.empty((max(cols, 1), ld), dtype=x.t.dtype, device=x.t.device).t()
    return _Opd(t.data_ptr(), ld, rows, cols, trans, t)


def _turn(x, trans):
    """op(x) stored with the given orientation: x itself, or a transposed copy."""
    if x.trans == trans:
        return x
    y = _like(x, x.cols, x.rows, trans)
    _copy(x.t[:x.rows, :x.cols], y.t[:y.rows, :y.cols])
    return y


def _copy(src, dst):
    ops.gecopy(src, dst, trans='T')


def _modified(*mats):
    for M in mats:
        if M is not None:
            M.storage.mark_local_modified(M.storage.origin_slot)


# -------------------------------------------------------------- distributed
def _grid_work(M, m, n, dtype=None):
    """A fresh m x n matrix with square tiles on M's grid."""
    slot = M.storage.origin_slot
    bc = M.storage.bc
    if bc.mb == bc.nb:
        return _fresh(M, m, n, slot, dtype)
    from ..core.matrix import Matrix
    s = M.storage
    W = Matrix(m, n, nb=bc.nb, p=bc.p, q=bc.q, comm=s.comm, dtype=dtype or s.dtype, device=s.device, order=bc.order)
    W.insertLocalTiles(device=s.device if slot == DEV else -1)
    return W


def _placed(X, W):
    """Does X store op(X) exactly where W stores its elements?"""
    return X._op == Op.NoTrans and X.global_offsets() == (0, 0) and _same_place(X, W)


def _onto(X, W):
    """X itself where it lies as W does, or a copy on W's grid (from offset 0)."""
    if _placed(X, W):
        return X
    F = _grid_work(W, X.m(), X.n(), X.storage.dtype)
    from ..parallel.redist import redistribute_pieces
    redistribute_pieces(X, F)
    return F


def _gather_k(X, W, rows):
    """This rank's rows of op(X), all columns (rows=True), or its columns, all
    rows: one broadcast per tile column (row) of X over the process row (column)."""
    F = _onto(X, W)
    grid, lb = grid_of(F), F.local_block()
    bc, dt, dev = F.storage.bc, F.storage.dtype, lb.data.device
    m, n, nb = F.m(), F.n(), bc.nb
    if rows:
        P = ops.colmajor_empty(lb.mloc, n, dt, dev)
        for k in range(-(-n // nb)):
            kb, lc = min(nb, n - k * nb), tiles_local_before(k, bc.q, bc.pc) * nb
            src = lb.data[:, lc:lc + kb] if k % bc.q == bc.pc else None
            if lb.mloc:
                P[:, k * nb:k * nb + kb].copy_(row_bcast(grid, src, k % bc.q, lb.mloc, kb, dt, dev))
    else:
        P = ops.colmajor_empty(m, lb.nloc, dt, dev)
        for k in range(-(-m // nb)):
            kb, lr = min(nb, m - k * nb), tiles_local_before(k, bc.p, bc.pr) * nb
            src = lb.data[lr:lr + kb, :] if k % bc.p == bc.pr else None
            if lb.nloc:
                P[k * nb:k * nb + kb, :].copy_(col_bcast(grid, src, k % bc.p, kb, lb.nloc, dt, dev))
    return _of_tensor(P, P.shape[0], P.shape[1])


def _vector(bias, mode, W):
    """This rank's part of a bias, as a dense vector operand."""
    F = _onto(bias, W)
    grid, lb = grid_of(F), F.local_block()
    dt, dev = F.storage.dtype, lb.data.device
    if mode == 1:
        mloc = W.local_block().mloc
        v = row_bcast(grid, lb.data if F.storage.bc.pc == 0 else None, 0, mloc, 1, dt, dev)
        return _of_tensor(v, mloc, 1)
    nloc = W.local_block().nloc
    v = col_bcast(grid, lb.data if F.storage.bc.pr == 0 else None, 0, 1, nloc, dt, dev)
    return _of_tensor(v, 1, nloc)


def _run_dist(mode, alpha, A, B, C, bias=None, bias_mode=0, act=0, beta=0.0, R=None, Z=()):
    """The product(s) on p x q ranks; every operand a Matrix on any grid."""
    W = []
    for c in C:
        bc = c.storage.bc
        W.append(c if bc.mb == bc.nb and _placed(c, c) and (not W or _placed(c, W[0]))
                 else _grid_work(W[0] if W else c, c.m(), c.n()))
    grid_rank = W[0].storage.bc.pr >= 0
    Zw = [None if z is None else (z if _placed(z, W[0]) else _grid_work(W[0], z.m(), z.n())) for z in Z]
    Rw = None if R is None or beta == 0 else _onto(R, W[0])
    if alpha != 0:
        As = [_gather_k(a, W[0], True) for a in A]
        Bs = [_gather_k(b, W[0], False) for b in B]
    else:
        lb = W[0].local_block()
        As, Bs = [_like(_opd(W[0]), lb.mloc, 0)], [_like(_opd(W[0]), 0, lb.nloc)]
    b = _NONE if bias is None else _vector(bias, bias_mode, W[0])
    if grid_rank:
        _launch(mode, alpha, As, Bs, [_opd(w) for w in W], b, bias_mode, act, beta,
                _NONE if Rw is None else _opd(Rw), [None if z is None else _opd(z) for z in Zw])
    _modified(*W, *Zw)
    for w, c in zip(list(W) + Zw, list(C) + list(Z)):
        if w is not None and w is not c:
            _copy_out(w, c)


# ------------------------------------------------------------------ products
def gemm_bias_act(alpha, A, B, bias, act, beta, R, C, Z=None, opts=None):
    """C = act(alpha op(A) op(B) + bias) + beta R.

    ``bias`` (or None) is m x 1, one value per row of C, or 1 x n, one per
    column.  ``act`` is an :class:`Activation` or its name ("identity", "relu",
    "gelu", "gelu_tanh", "silu").  ``R`` (or None) is the residual; it may be C
    itself and is not read when beta = 0; A and B are not read when alpha = 0.
    ``Z`` (or None) receives the argument of act, which
    :func:`gemm_bias_act_grad` takes.  C and Z overlap no other matrix of the
    call."""
    a = _act(act)
    if C._op != Op.NoTrans:
        gemm_bias_act(alpha, _t(B), _t(A), _t(bias), act, beta, _t(R), _t(C), _t(Z), opts)
        return C
    m, n, k = C.m(), C.n(), A.n()
    bshape, bmode = _bias_shape(bias, m, n, "gemm_bias_act")
    mats = dict(A=A, B=B, bias=bias, R=R, C=C, Z=Z)
    _check(mats, dict(A=(m, k), B=(k, n), bias=bshape, R=(m, n), C=(m, n), Z=(m, n)), "gemm_bias_act")
    with trace_block("gemm_bias_act"):
        if not _single(*(M for M in mats.values() if M is not None)):
            _run_dist(PLAIN, alpha, [A], [B], [C], bias, bmode, a, beta, R, (Z,))
            return C
        oa, ob, oc = _opd(A, "A"), _opd(B, "B"), _opd(C, "C")
        o1, orr = (_NONE if bias is None else _opd(bias, "bias")), (_NONE if R is None else _opd(R, "R"))
        oz = _NONE if Z is None else _opd(Z, "Z")
        _outputs([oc, oz], [oa, ob, o1, orr], ("C", "Z"), ("A", "B", "bias", "R"), {(0, 3)})
        with _on(oc.t):
            # transposed views of R and Z go through workspace
            r2 = orr if orr.t is None or beta == 0 else _turn(orr, False)
            z2 = _like(oz, m, n) if oz.trans else oz
            _launch(PLAIN, alpha, [oa], [ob], [oc], o1, bmode, a, beta, r2, (z2 if z2.t is not None else None,))
            if z2 is not oz:
                _copy(z2.t[:m, :n], oz.t[:oz.rows, :oz.cols])
        _modified(C, Z)
    return C


def gemm_gated(A1, A2, B, act, C, Z1=None, Z2=None, opts=None):
    """C = act(op(A1) op(B)) o (op(A2) op(B)), o elementwise: the gated
    projection of a feed-forward block, both products and their combination in
    one kernel.

    A1 and A2 enter with the same op.  ``Z1``, ``Z2`` (or None) receive the two
    products, which :func:`gemm_gated_grad` takes.  C, Z1 and Z2 overlap no
    other matrix of the call."""
    a = _act(act)
    m, n, k = C.m(), C.n(), A1.n()
    mats = dict(A1=A1, A2=A2, B=B, C=C, Z1=Z1, Z2=Z2)
    _check(mats, dict(A1=(m, k), A2=(m, k), B=(k, n), C=(m, n), Z1=(m, n), Z2=(m, n)), "gemm_gated")
    with trace_block("gemm_gated"):
        if not _single(*(M for M in mats.values() if M is not None)):
            outs = [M if M is None or M._op == Op.NoTrans else _grid_work(M, m, n) for M in (C, Z1, Z2)]
            _run_dist(GATED, 1.0, [A1, A2], [B], outs[:1], act=a, Z=tuple(outs[1:]))
            for w, M in zip(outs, (C, Z1, Z2)):
                if w is not M:
                    _copy_out(w, M)
            return C
        o1, o2, ob, oc = _opd(A1, "A1"), _opd(A2, "A2"), _opd(B, "B"), _opd(C, "C")
        z1, z2 = (_NONE if Z is None else _opd(Z, "Z") for Z in (Z1, Z2))
        _outputs([oc, z1, z2], [o1, o2, ob], ("C", "Z1", "Z2"), ("A1", "A2", "B"))
        with _on(oc.t):
            if o1.trans != o2.trans:
                o2 = _turn(o2, o1.trans)
            # a transposed output is made in workspace and copied
            w = [x if x.t is None or not x.trans else _like(x, m, n) for x in (oc, z1, z2)]
            _launch(GATED, 1.0, [o1, o2], [ob], w[:1], act=a, Z=[x if x.t is not None else None for x in w[1:]])
            for x, y in zip(w, (oc, z1, z2)):
                if x is not y:
                    _copy(x.t[:m, :n], y.t[:y.rows, :y.cols])
        _modified(C, Z1, Z2)
    return C


# ----------------------------------------------------------------- gradients
def _act_grad(m, n, act, dC, Z1, Z2, dZ1, dZ2, db=_NONE, bias_mode=0, wide=False):
    """One rank's elementwise pass; operands not transposed."""
    t = dC.t
    if m == 0 or n == 0:
        if db.t is not None:
            db.t.zero_()
        return
    mod, dt = kmod(t), REAL_CODE[t.dtype]
    nbytes = mod.act_grad_ws(dt, bias_mode, m, n)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=t.device) if nbytes else None
    mod.act_grad(dt, m, n, act, dC.ptr, dC.ld, Z1.ptr, Z1.ld, Z2.ptr, Z2.ld, dZ1.ptr, dZ2.ptr, dZ1.ld,
                 db.ptr, _inc(db), bias_mode, wide, 0 if ws is None else ws.data_ptr(), raw_stream(t))


def gemm_bias_act_grad(alpha, A, B, act, Z, dC, dA, dB, dbias, opts=None):
    """Gradients of :func:`gemm_bias_act` with respect to A, B and bias:

        dZ = dC o act'(Z),  dA = alpha dZ op(B)^T,  dB = alpha op(A)^T dZ,
        dbias = row sums of dZ (column sums where dbias is 1 x n)

    dA and dB have the shapes of op(A) and op(B) (pass a transposed view for an
    operand that entered transposed); None leaves a gradient out.  ``Z`` is what
    the forward pass stored (may be None for the identity).  The residual's
    gradient is beta dC.  dZ is rounded to the matrices' type between the two
    steps, the bias gradient is summed from its unrounded values."""
    what = "gemm_bias_act_grad"
    a = _act(act)
    m, n, k = dC.m(), dC.n(), A.n()
    bshape, bmode = _bias_shape(dbias, m, n, what)
    if Z is None and a:
        raise SlateError(f"{what}: Z is wanted for activation {act}")
    mats = dict(A=A, B=B, Z=Z, dC=dC, dA=dA, dB=dB, dbias=dbias)
    _check(mats, dict(A=(m, k), B=(k, n), Z=(m, n), dC=(m, n), dA=(m, k), dB=(k, n), dbias=bshape), what)
    Z = Z if a else None
    with trace_block(what):
        if not _single(*(M for M in mats.values() if M is not None)):
            dZ = _dz_dist(a, dC, (Z, None), dbias, bmode)[0]
            if dA is not None:
                _run_dist_any(PLAIN, alpha, [dZ], [_t(B)], [dA])
            if dB is not None:
                _run_dist_any(PLAIN, alpha, [_t(A)], [dZ], [dB])
            return
        oa, ob, oz, oc, ga, gb, gv = (_NONE if M is None else _opd(M, s) for M, s in
                                      zip((A, B, Z, dC, dA, dB, dbias), ("A", "B", "Z", "dC", "dA", "dB", "dbias")))
        _outputs([ga, gb, gv], [oa, ob, oz, oc], ("dA", "dB", "dbias"), ("A", "B", "Z", "dC"))
        with _on(oc.t):
            dZ = oc
            if a or dbias is not None:
                oz = oz if oz.t is None else _turn(oz, oc.trans)
                dZ = _like(oc, oc.rows, oc.cols, oc.trans) if a and (dA is not None or dB is not None) else _NONE
                mode = bmode if not oc.trans or not bmode else 3 - bmode
                _act_grad(oc.rows, oc.cols, a, oc, oz, _NONE, dZ, _NONE, gv, mode)
                dZ = dZ if a else oc
            if dA is not None:
                _product(PLAIN, alpha, [dZ], [ob.T], [ga])
            if dB is not None:
                _product(PLAIN, alpha, [oa.T], [dZ], [gb])
        _modified(dA, dB, dbias)


def _product(mode, alpha, A, B, C):
    """One rank's product(s) into outputs of either orientation."""
    if C[0].trans:
        A, B, C = [x.T for x in B], [x.T for x in A], [x.T for x in C]
    _launch(mode, alpha, A, B, C)


def gemm_gated_grad(A1, A2, B, act, Z1, Z2, dC, dA1, dA2, dB, opts=None):
    """Gradients of :func:`gemm_gated`:

        dZ1 = dC o Z2 o act'(Z1),  dZ2 = dC o act(Z1),
        dA1 = dZ1 op(B)^T,  dA2 = dZ2 op(B)^T,  dB = op(A1)^T dZ1 + op(A2)^T dZ2

    with Z1, Z2 as the forward pass stored them; None leaves a gradient out.
    Both weight gradients are one launch, and dB is one sum over both products,
    rounded once."""
    what = "gemm_gated_grad"
    a = _act(act)
    m, n, k = dC.m(), dC.n(), A1.n()
    mats = dict(A1=A1, A2=A2, B=B, Z1=Z1, Z2=Z2, dC=dC, dA1=dA1, dA2=dA2, dB=dB)
    if Z1 is None or Z2 is None:
        raise SlateError(f"{what}: Z1 and Z2 are wanted")
    w, z = (m, k), (m, n)
    _check(mats, dict(A1=w, A2=w, B=(k, n), Z1=z, Z2=z, dC=z, dA1=w, dA2=w, dB=(k, n)), what)
    with trace_block(what):
        if not _single(*(M for M in mats.values() if M is not None)):
            dZ = _dz_dist(a, dC, (Z1, Z2), None, 0)
            for d, g in zip(dZ, (dA1, dA2)):
                if g is not None:
                    _run_dist_any(PLAIN, 1.0, [d], [_t(B)], [g])
            if dB is not None:
                _run_dist_any(SUM, 1.0, [_t(A1), _t(A2)], dZ, [dB])
            return
        names = ("A1", "A2", "B", "Z1", "Z2", "dC", "dA1", "dA2", "dB")
        o1, o2, ob, z1, z2, oc, g1, g2, gb = (_NONE if M is None else _opd(M, s) for M, s in zip(mats.values(), names))
        _outputs([g1, g2, gb], [o1, o2, ob, z1, z2, oc], names[6:], names[:6])
        with _on(oc.t):
            d1, d2 = _like(oc, oc.rows, oc.cols, oc.trans), _like(oc, oc.rows, oc.cols, oc.trans)
            _act_grad(oc.rows, oc.cols, a, oc, _turn(z1, oc.trans), _turn(z2, oc.trans), d1, d2)
            if dA1 is not None and dA2 is not None and g1.trans == g2.trans:
                _product(PAIR, 1.0, [d1, d2], [ob.T, ob.T], [g1, g2])
            else:
                for d, g in ((d1, g1), (d2, g2)):
                    if g.t is not None:
                        _product(PLAIN, 1.0, [d], [ob.T], [g])
            if dB is not None:
                _product(SUM, 1.0, [o1.T, (o2 if o2.trans == o1.trans else _turn(o2, o1.trans)).T], [d1, d2], [gb])
        _modified(dA1, dA2, dB)


def _run_dist_any(mode, alpha, A, B, C):
    """_run_dist into outputs of either orientation."""
    if C[0]._op != Op.NoTrans:
        A, B, C = [_t(x) for x in B], [_t(x) for x in A], [_t(x) for x in C]
    _run_dist(mode, alpha, A, B, C)


def _dz_dist(act, dC, Z, dbias, bmode):
    """dZ (one or two matrices, from offset 0 on dC's grid) and the bias
    gradient: local sums in 32 (64) bits, one all-reduce over the process row
    (column), one rounding."""
    W = dC if dC.storage.bc.mb == dC.storage.bc.nb and _placed(dC, dC) else None
    if W is None:
        W = _grid_work(dC, dC.m(), dC.n())
        from ..parallel.redist import redistribute_pieces
        redistribute_pieces(dC, W)
    Zw = [None if z is None else _onto(z, W) for z in Z]
    two = Zw[1] is not None
    dZ = [_grid_work(W, dC.m(), dC.n()) for _ in range(2 if two else 1)] if act or two else [W]
    lb, s = W.local_block(), W.storage
    db, sums = _NONE, None
    if dbias is not None:
        wide = torch.float64 if s.dtype == torch.float64 else torch.float32
        sums = torch.zeros(lb.mloc if bmode == 1 else lb.nloc, dtype=wide, device=lb.data.device)
        db = _Opd(sums.data_ptr(), 1, sums.numel(), 1, False, sums)
    if s.bc.pr >= 0 and (act or two or dbias is not None):
        oz = [_NONE if z is None else _opd(z) for z in Zw]
        od = [_opd(d) for d in dZ] if act or two else [_NONE]
        _act_grad(lb.mloc, lb.nloc, act, _opd(W), oz[0], oz[1], od[0], od[1] if two else _NONE, db, bmode, True)
    if act or two:
        _modified(*dZ)
    if dbias is not None:
        grid = grid_of(W)
        comm = grid.row_comm if bmode == 1 else grid.col_comm
        if s.bc.pr >= 0 and comm.size > 1 and sums.numel():
            comm.allreduce(sums, "sum")
        V = _grid_work(W, dbias.m(), dbias.n())
        lv = V.local_block()
        if lv.mloc and lv.nloc:
            ops.gecopy(sums.view(-1, 1) if bmode == 1 else sums.view(1, -1), lv.data)
        _modified(V)
        _copy_out(V, dbias)
    return dZ


# ------------------------------------------------------------------ clipping
def _clip_views(mats, what):
    if not isinstance(mats, (list, tuple)):
        raise SlateError(f"{what}: a list of matrices is wanted")
    out, first = [], None
    for M in mats:
        s = M.storage
        if getattr(M, "_kind", "general") != "general" or s.bc is None:
            raise SlateError(f"{what}: general block-cyclic matrices are wanted")
        if s.origin_slot is None:
            raise SlateError(f"{what}: a matrix has no tiles (insertLocalTiles)")
        if first is None:
            first = s
        elif s.dtype != first.dtype or _where(s) != _where(first):
            raise SlateError(f"{what}: the matrices differ in type or device ({s.dtype} on {_where(s)}, "
                             f"{first.dtype} on {_where(first)})")
        elif s.comm is not first.comm and s.comm.ranks != first.comm.ranks:
            raise SlateError(f"{what}: the matrices differ in communicator")
        out.append(_opd(M))
    return out, first


def clip_norm(max_norm, A, B=None, opts=None):
    """B_i = min(1, max_norm / s) A_i with s the Frobenius norm of all matrices
    of the list A together; returns s as a float64 tensor on the matrices'
    device (no host synchronisation).

    B = None scales in place.  B's matrices have A's shapes and distribution,
    and A's type or, for 16-bit A, float32.  Where s is not finite the matrices
    are copied (left) as they are, so that a caller can look at s and skip the
    step.  The squares are summed in 64 bits, in an order that depends on the
    sizes alone.  Matrices written overlap no other matrix of the call, except
    that B_i may be A_i."""
    what = "clip_norm"
    limit = float(max_norm)
    if not limit >= 0:
        raise SlateError(f"{what}: max_norm {max_norm} is not >= 0")
    return _clip(what, limit, A, A if B is None else B)


def global_norm(A, opts=None):
    """Frobenius norm of all matrices of the list A together (a float: waits
    for the device, as ``norm`` does)."""
    return float(_clip("global_norm", None, A, A))


def _clip(what, limit, A, B):
    va, s = _clip_views(A, what)
    if not va:
        return torch.zeros((), dtype=torch.float64)
    vb, sb = (va, s) if B is A else _clip_views(B, what)
    cplx = {torch.complex64: torch.float32, torch.complex128: torch.float64}
    ta, tb = cplx.get(s.dtype, s.dtype), cplx.get(sb.dtype, sb.dtype)
    if ta not in REAL_CODE or not (s.dtype == sb.dtype or (_BYTES[ta] == 2 and sb.dtype == torch.float32)):
        raise SlateError(f"{what}: no scaling from {s.dtype} to {sb.dtype}")
    if len(vb) != len(va) or _where(sb) != _where(s):
        raise SlateError(f"{what}: B has {len(vb)} matrices on {_where(sb)}, A has {len(va)} on {_where(s)}")
    two = 2 if s.dtype in cplx else 1
    with trace_block(what):
        if vb is not va:
            for X, Y, x, y in zip(A, B, va, vb):
                if X._op != Y._op or (x.rows, x.cols) != (y.rows, y.cols) or X.m() != Y.m() or X.n() != Y.n() or \
                        (s.comm.size > 1 and not _same_place(X, Y)):
                    raise SlateError(f"{what}: B's matrices want the shapes, ops and distribution of A's")
        if limit is not None:
            seen = set()
            for y in vb:
                if y.rows and y.cols:
                    if y.ptr in seen:
                        raise SlateError(f"{what}: a matrix is in the list twice")
                    seen.add(y.ptr)
        t = va[0].t
        mod, st = kmod(t), raw_stream(t)
        list_ = [(x.ptr, x.ld * two, y.ptr, y.ld * two, x.rows * two, x.cols) for x, y in zip(va, vb)]
        with _on(t):
            ws = torch.empty(mod.clip_ws(list_) + 4, dtype=torch.float64, device=t.device)
            base = ws.data_ptr()
            part = base + 32
            norm = ws[0]
            n = mod.clip_sum(REAL_CODE[ta], list_, part, st)
            if s.comm.size > 1:
                mod.clip_join(part, n, base + 8, st)
                s.comm.allreduce(ws[1:4], "sum")
                part, n = base + 8, 1
            mod.clip_scale(REAL_CODE[ta], REAL_CODE[tb], list_, 0.0 if limit is None else limit, part, n, base,
                           limit is not None, st)
        if limit is not None:
            _modified(*B)
    return norm


def _same_place(X, Y):
    """The same tiles of the same grid, from the same offset (the shapes may differ)."""
    a, b = X.storage.bc, Y.storage.bc
    return (a.mb, a.nb, a.p, a.q, a.order) == (b.mb, b.nb, b.p, b.q, b.order) and \
        X.global_offsets() == Y.global_offsets() and X.storage.comm.ranks == Y.storage.comm.ranks

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
synchronise, and can be captured into a hipGraph (on one rank).  On p x q ranks
the products wait once where matrices over buffers of the caller are written or
stand beside written ones: the ranks agree on whether any of these overlap.
"""
from __future__ import annotations

import torch

from .. import ops
from .._native import REAL_CODE, kmod, raw_stream
from ..core.enums import Activation, Op, Option
from ..core.exceptions import SlateError
from ..core.options import get_option
from ..core.storage import DEV, debug_checks
from ..utils.trace import trace_block
from ._panels import col_bcast, row_bcast
from ._util import grid_of, tiles_local_before
from .blas3 import _copy_out, _fresh

PLAIN, GATED, SUM, PAIR = 0, 1, 2, 3
_ACT = {a: i for i, a in enumerate(Activation)}
_ACT.update({a.name.lower(): i for a, i in list(_ACT.items())})
_BYTES = {torch.bfloat16: 2, torch.float16: 2, torch.float32: 4, torch.float64: 8, torch.complex64: 8, torch.complex128: 16}


_HALF = (torch.bfloat16, torch.float16)
_DEVICES = {}          # one object per device, so that operands compare them by identity


# ------------------------------------------------------------------ operands
class _Opd:
    """One rank's strided column-major operand: first and one past the last
    address, leading dimension, stored and logical shape, whether it enters
    transposed, and the tensor that owns it.  That of a view: the tile table of
    its storage and the version at which it was whole."""

    __slots__ = ("ptr", "end", "ld", "rows", "cols", "m", "n", "trans", "t", "dt", "dev", "table", "version")

    def __init__(self, ptr, ld, rows, cols, trans, t):
        self.dt, self.dev = (None, None) if t is None else (t.dtype, _DEVICES.setdefault(t.device, t.device))
        self.ptr, self.ld, self.rows, self.cols, self.trans, self.t = ptr, ld, rows, cols, trans, t
        self.m, self.n = (cols, rows) if trans else (rows, cols)
        self.end = ptr + ((cols - 1) * ld + rows) * _BYTES[t.dtype] if rows and cols else ptr

    @property
    def T(self):
        return _Opd(self.ptr, self.ld, self.rows, self.cols, not self.trans, self.t)

    @property
    def op(self):
        return 'T' if self.trans else 'N'


_NONE = _Opd(0, 0, 0, 0, False, None)


def _of_tensor(t, rows, cols, trans=False, name="matrix"):
    if cols > 1:
        ld = t.stride(1)
        if ld < rows:
            raise SlateError(f"{name}: columns overlap (leading dimension {ld} < {rows} rows)")
    else:
        ld = rows + 7 & -8 or 8            # of no meaning: any aligned one
    return _Opd(t.data_ptr(), ld, rows, cols, trans, t)


def _opd(M, name="matrix"):
    """The (one) rank's operand of a view.  A view remembers it, and uses it again
    while it has the same storage, no state of whose tiles has changed (new buffers
    and writes on the other side do), and its buffer is at the same place.  (With
    the debug checks on, prepare_local runs them on every call.)"""
    s = M.storage
    x = M.__dict__.get("_operand")
    if x is not None and x.table is s.table and x.version == s.table.version() and x.t.data_ptr() == x.ptr \
            and not debug_checks():
        return x
    slot = s.origin_slot
    if M._mt == s.mt and M._nt == s.nt and not (M.row0_offset or M.col0_offset) and M.last_mb is None \
            and M.last_nb is None and slot is not None:
        t, rows, cols = s.prepare_local(slot), s.bc.mloc, s.bc.nloc
    else:
        t = M.local_block().data
        rows, cols = t.shape
    x = _of_tensor(t, rows, cols, M._op is not Op.NoTrans, name)
    x.table = s.table
    x.version = s._valid.get(s.origin_slot, -1)      # (an older one is never met again)
    M.__dict__["_operand"] = x
    return x


def _operands(what, names, mats):
    """Operands of a one-rank call's matrices (None stays none): one element
    type, one device, general block-cyclic storage."""
    out, first = [], None
    for name, M in zip(names, mats):
        if M is None:
            out.append(_NONE)
            continue
        s = M.storage
        if not M._whole or s.bc is None:
            raise SlateError(f"{what}: {name} must be a general block-cyclic matrix")
        if s.origin_slot is None:
            raise SlateError(f"{what}: {name} has no tiles (insertLocalTiles)")
        x = _opd(M, name)
        if first is None:
            first, dt, dev = x, x.dt, x.dev
            if dt not in REAL_CODE:
                raise SlateError(f"{what}: element type {dt} (bfloat16, float16, float32 or float64 are wanted)")
        elif x.dt is not dt:
            raise SlateError(f"{what}: {name} has type {x.dt}, the others {dt}")
        elif x.dev is not dev:
            raise SlateError(f"{what}: {name} is on {x.dev}, the others on {dev}")
        out.append(x)
    return out


def _one(mats):
    """1: every matrix is this rank's alone; 2: each is on one rank, some among
    several; 0: some is on several."""
    one = 1
    for M in mats:
        if M is not None:
            s = M.storage
            if s.bc is None:
                return 1                    # not block-cyclic: the checks refuse it
            if s.comm.size > 1:
                if s.bc.p * s.bc.q > 1:
                    return 0
                one = 2
    return one


def _shape(what, name, x, m, n):
    if x.t is not None and (x.m != m or x.n != n):
        raise SlateError(f"{what}: {name} is {x.m} x {x.n}, {m} x {n} is wanted")


def _t(M):
    """Transposed view (the element types are real: ConjTrans is Trans)."""
    return None if M is None else M._clone(_op=Op.NoTrans if M._op != Op.NoTrans else Op.Trans)


def _overlap(x, y):
    """Do two operands share elements?  Blocks of one leading dimension are
    compared as rectangles, others by their address ranges."""
    if x.end <= y.ptr or y.end <= x.ptr:
        return False
    es, off = _BYTES[x.t.dtype], y.ptr - x.ptr
    if y.t.dtype != x.t.dtype or off % es or (x.cols > 1 and y.cols > 1 and x.ld != y.ld):
        return True
    ld = x.ld if x.cols > 1 else y.ld
    if x.rows > ld or y.rows > ld:
        return True
    dc, dr = divmod(off // es, ld)
    for c, r in ((dc, dr), (dc + 1, dr - ld)):
        if r < x.rows and -r < y.rows and c < x.cols and -c < y.cols:
            return True
    return False


def _outputs(what, outs, ins, same=None):
    """Outputs [(name, operand)] share no element with each other or with
    inputs; ``same`` names an input that the first output may be (the same view:
    each element is read, then written, by one thread)."""
    for i, (nx, x) in enumerate(outs):
        if x.t is None:
            continue
        lo, hi = x.ptr, x.end
        for ny, y in ins:
            if y.ptr < hi and lo < y.end and not (i == 0 and ny == same and (x.ptr, x.ld, x.trans) == (y.ptr, y.ld, y.trans)) \
                    and _overlap(x, y):
                raise SlateError(f"{what}: output {nx} overlaps {ny}")
        for ny, y in outs[:i]:
            if y.ptr < hi and lo < y.end and _overlap(x, y):
                raise SlateError(f"{what}: outputs {nx} and {ny} overlap")


def _rect(M):
    """A view's block of its storage: first row and column, one past the last ones."""
    r, c = M.global_offsets()
    return r, c, r + M._um(), c + M._un()


def _share(X, Y, may):
    """Do two views of one storage share elements?  may: they may be the same view."""
    a, b = _rect(X), _rect(Y)
    if may and a == b and (X._op is Op.NoTrans) == (Y._op is Op.NoTrans):
        return False
    return max(a[0], b[0]) < min(a[2], b[2]) and max(a[1], b[1]) < min(a[3], b[3])


def _apart(what, outs, ins, same=None, ask=True):
    """:func:`_outputs` for matrices [(name, M)] on a grid of ranks, with one
    verdict on every rank: views of one storage are compared by their global
    indexes.  Buffers of the caller are compared by the addresses on this rank;
    then (ask) the ranks tell each other, and the call waits for the device."""
    found = comm = None
    for i, (nx, X) in enumerate(outs):
        if X is None:
            continue
        for ny, Y in ins + outs[:i]:
            if Y is None:
                continue
            may = i == 0 and ny == same
            if X.storage is Y.storage:
                if _share(X, Y, may):
                    raise SlateError(f"{what}: output {nx} overlaps {ny}")
            elif ask and (X.storage.wraps or Y.storage.wraps):
                comm = X.storage.comm
                x, y = _opd(X), _opd(Y)
                if not (may and (x.ptr, x.ld, x.trans) == (y.ptr, y.ld, y.trans)) and _overlap(x, y):
                    found = found or f"output {nx} overlaps {ny}"
    if comm is not None and comm.allreduce_scalar(float(found is not None), "max"):
        raise SlateError(f"{what}: {found or 'an output overlaps another matrix on another rank'}")


def _act(act):
    """Kernel code of an Activation, its name or its character."""
    try:
        return _ACT[act]
    except (KeyError, TypeError):
        try:
            return _ACT[Activation.from_string(act)]
        except ValueError:
            raise SlateError(f"unknown activation {act!r}") from None


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
        if not M._whole or s.bc is None:
            raise SlateError(f"{what}: {name} must be a general block-cyclic matrix")
        if first is None:
            first = s
            if s.dtype not in REAL_CODE:
                raise SlateError(f"{what}: element type {s.dtype} (bfloat16, float16, float32 or float64 are wanted)")
        elif s.dtype != first.dtype:
            raise SlateError(f"{what}: {name} has type {s.dtype}, the others {first.dtype}")
        elif s.comm.ranks != first.comm.ranks:
            raise SlateError(f"{what}: {name} has another communicator than the others")
        if s.origin_slot is None:
            raise SlateError(f"{what}: {name} has no tiles (insertLocalTiles)")
        if _where(s) != _where(first):
            raise SlateError(f"{what}: {name} is on {_where(s)}, the others on {_where(first)}")
        m, n = shapes[name]
        if M.m() != m or M.n() != n:
            raise SlateError(f"{what}: {name} is {M.m()} x {M.n()}, {m} x {n} is wanted")
    return first


def _bias_mode(what, shape, m, n):
    """1: one value per row (m x 1), 2: per column (1 x n), 0: no bias."""
    if shape is None:
        return 0
    if shape == (m, 1):
        return 1
    if shape == (1, n):
        return 2
    raise SlateError(f"{what}: bias is {shape[0]} x {shape[1]}, {m} x 1 or 1 x {n} is wanted")


def _bias_of(what, bias, m, n):
    """(shape to check, mode) of a distributed bias."""
    mode = _bias_mode(what, None if bias is None else (bias.m(), bias.n()), m, n)
    return ((1, n) if mode == 2 else (m, 1)), mode


def _inc(b):
    """Distance of a vector operand's elements."""
    return 1 if b.rows > 1 or b.cols <= 1 else b.ld


_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


class _on:
    """The operands' device made current (launches and workspaces go there)."""

    def __init__(self, t):
        self.ctx = None
        if t.is_cuda and t.device.index != _current_device():
            self.ctx = torch.cuda.device(t.device)

    def __enter__(self):
        if self.ctx is not None:
            self.ctx.__enter__()

    def __exit__(self, *e):
        if self.ctx is not None:
            self.ctx.__exit__(*e)


def _launch(mode, alpha, A1, A2, B1, B2, C1, C2, bias=_NONE, bias_mode=0, act=0, beta=0.0, R=_NONE, Z1=_NONE, Z2=_NONE,
            more=()):
    """One rank's product(s); outputs, R and Z not transposed; more: the third and
    fourth operands (A, B) of a sum."""
    t = C1.t
    m, n, k = C1.rows, C1.cols, A1.n
    if m == 0 or n == 0:
        return
    if alpha == 0:
        k = 0                                   # op(A) op(B) is not read
    if beta == 0:
        R = _NONE
    if ops._FLOPS is not None:
        ops._FLOPS[0] += 2 * m * n * k * (1 if mode == PLAIN else 2 + len(more))
    call = kmod(t).gemm_act
    args = (REAL_CODE[t.dtype], mode, A1.op, B1.op, m, n, k, alpha, A1.ptr, A1.ld, A2.ptr, A2.ld, B1.ptr, B1.ld,
            B2.ptr, B2.ld, C1.ptr, C1.ld, C2.ptr, C2.ld, bias.ptr, _inc(bias), bias_mode, act, beta, R.ptr, R.ld,
            Z1.ptr, Z1.ld, Z2.ptr, Z2.ld, [i for a, b in more for i in (a.ptr, a.ld, b.ptr, b.ld)])
    st = raw_stream(t)
    nbytes = call(*args, 0, st)
    if nbytes:                                  # few tiles: partial sums of pieces of k
        ws = torch.empty(nbytes, dtype=torch.uint8, device=t.device)
        call(*args, ws.data_ptr(), st)


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
        # (the terms of a sum may share operands: each is gathered once)
        As = {id(a): _gather_k(a, W[0], True) for a in {id(a): a for a in A}.values()}
        Bs = {id(b): _gather_k(b, W[0], False) for b in {id(b): b for b in B}.values()}
        As, Bs = [As[id(a)] for a in A], [Bs[id(b)] for b in B]
    else:
        lb = W[0].local_block()
        As, Bs = [_like(_opd(W[0]), lb.mloc, 0)], [_like(_opd(W[0]), 0, lb.nloc)]
    b = _NONE if bias is None else _vector(bias, bias_mode, W[0])
    if grid_rank:
        more = list(zip(As[2:], Bs[2:]))
        As, Bs, Ws = ((x + [_NONE])[:2] for x in (As, Bs, [_opd(w) for w in W]))
        with _on(Ws[0].t):
            _launch(mode, alpha, *As, *Bs, *Ws, b, bias_mode, act, beta, _NONE if Rw is None else _opd(Rw),
                    *[_NONE if z is None else _opd(z) for z in Zw], more=more)
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
    what, mats = "gemm_bias_act", (A, B, bias, R, C, Z)
    with trace_block(what):
        one = _one(mats)
        if one != 1:
            m, n, k = C.m(), C.n(), A.n()
            bshape, bmode = _bias_of(what, bias, m, n)
            _check(dict(A=A, B=B, bias=bias, R=R, C=C, Z=Z),
                   dict(A=(m, k), B=(k, n), bias=bshape, R=(m, n), C=(m, n), Z=(m, n)), what)
            _apart(what, [("C", C), ("Z", Z)], [("A", A), ("B", B), ("bias", bias), ("R", R)], "R", not one)
            if not one:
                _run_dist(PLAIN, alpha, [A], [B], [C], bias, bmode, a, beta, R, (Z,))
            if not one or C.storage.bc.pr < 0:
                return C
        oa, ob, o1, orr, oc, oz = _operands(what, ("A", "B", "bias", "R", "C", "Z"), mats)
        m, n, k = oc.m, oc.n, oa.n
        _shape(what, "A", oa, m, k)
        _shape(what, "B", ob, k, n)
        _shape(what, "R", orr, m, n)
        _shape(what, "Z", oz, m, n)
        bmode = _bias_mode(what, None if bias is None else (o1.m, o1.n), m, n)
        _outputs(what, (("C", oc), ("Z", oz)), (("A", oa), ("B", ob), ("bias", o1), ("R", orr)), "R")
        with _on(oc.t):
            # transposed views of R and Z go through workspace
            r2 = _turn(orr, False) if orr.trans and beta != 0 else orr
            z2 = _like(oz, m, n) if oz.trans else oz
            _launch(PLAIN, alpha, oa, _NONE, ob, _NONE, oc, _NONE, o1, bmode, a, beta, r2, z2)
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
    what, mats = "gemm_gated", (A1, A2, B, C, Z1, Z2)
    with trace_block(what):
        one = _one(mats)
        if one != 1:
            m, n, k = C.m(), C.n(), A1.n()
            _check(dict(A1=A1, A2=A2, B=B, C=C, Z1=Z1, Z2=Z2),
                   dict(A1=(m, k), A2=(m, k), B=(k, n), C=(m, n), Z1=(m, n), Z2=(m, n)), what)
            _apart(what, [("C", C), ("Z1", Z1), ("Z2", Z2)], [("A1", A1), ("A2", A2), ("B", B)], None, not one)
            if not one:
                outs = [M if M is None or M._op == Op.NoTrans else _grid_work(M, m, n) for M in (C, Z1, Z2)]
                _run_dist(GATED, 1.0, [A1, A2], [B], outs[:1], act=a, Z=tuple(outs[1:]))
                for w, M in zip(outs, (C, Z1, Z2)):
                    if w is not M:
                        _copy_out(w, M)
            if not one or C.storage.bc.pr < 0:
                return C
        o1, o2, ob, oc, z1, z2 = _operands(what, ("A1", "A2", "B", "C", "Z1", "Z2"), mats)
        m, n, k = oc.m, oc.n, o1.n
        _shape(what, "A1", o1, m, k)
        _shape(what, "A2", o2, m, k)
        _shape(what, "B", ob, k, n)
        _shape(what, "Z1", z1, m, n)
        _shape(what, "Z2", z2, m, n)
        _outputs(what, (("C", oc), ("Z1", z1), ("Z2", z2)), (("A1", o1), ("A2", o2), ("B", ob)))
        with _on(oc.t):
            if o1.trans != o2.trans:
                o2 = _turn(o2, o1.trans)
            # a transposed output is made in workspace and copied
            w = [_like(x, m, n) if x.trans else x for x in (oc, z1, z2)]
            _launch(GATED, 1.0, o1, o2, ob, _NONE, w[0], _NONE, _NONE, 0, a, 0.0, _NONE, w[1], w[2])
            for x, y in zip(w, (oc, z1, z2)):
                if x is not y:
                    _copy(x.t[:m, :n], y.t[:y.rows, :y.cols])
        _modified(C, Z1, Z2)
    return C


# ----------------------------------------------------------------- gradients
def _act_grad(m, n, act, dC, Z1, Z2, dZ1, dZ2, db=_NONE, bias_mode=0, wide=False, rest=(_NONE, _NONE)):
    """One rank's elementwise pass; operands not transposed; rest: for what the
    rounding of dZ1 and dZ2 leaves over."""
    t = dC.t
    if m == 0 or n == 0:
        if db.t is not None:
            db.t[:db.rows, :db.cols].zero_()
        return
    mod, dt = kmod(t), REAL_CODE[t.dtype]
    nbytes = mod.act_grad_ws(dt, bias_mode, m, n)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=t.device) if nbytes else None
    mod.act_grad(dt, m, n, act, dC.ptr, dC.ld, Z1.ptr, Z1.ld, Z2.ptr, Z2.ld, dZ1.ptr, dZ2.ptr,
                 rest[0].ptr, rest[1].ptr, dZ1.ld, db.ptr, _inc(db), bias_mode, wide, 0 if ws is None else ws.data_ptr(), raw_stream(t))


class _Made:
    """Stands for a dZ, or what its rounding leaves over, in the workspace of :func:`_grad_run`."""
    __slots__ = ("ptr", "ld")

    def __init__(self, ptr):
        self.ptr, self.ld = ptr, 0


_DZ = [_Made(-1 - i) for i in range(4)]


def _step(steps, mode, k, A, at, B, bt, c, c2=_NONE):
    """Adds products op(A_i) op(B_i) into c, of either orientation, to steps; at
    and bt: do the operands enter transposed?"""
    if c.t is None:
        return
    if ops._FLOPS is not None:
        ops._FLOPS[0] += 2 * c.rows * c.cols * k * len(A)
    if c.trans:
        A, at, B, bt = B, not bt, A, not at
    steps += (mode, at, bt, c.rows, c.cols, k)
    fill = [0, 0] * (steps[14] - len(A))
    for x in A:
        steps += (x.ptr, x.ld)
    steps += fill
    for x in B:
        steps += (x.ptr, x.ld)
    steps += fill
    steps += (c.ptr, c.ld, c2.ptr, c2.ld)


def _grad_run(alpha, oc, steps):
    """One rank's backward pass on the device as two calls: its workspace, itself."""
    t = oc.t
    code, st, call = REAL_CODE[t.dtype], raw_stream(t), kmod(t).ffn_grad
    nbytes = call(code, alpha, steps, 0, st)
    ws = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=t.device)
    call(code, alpha, steps, ws.data_ptr(), st)


def gemm_bias_act_grad(alpha, A, B, act, Z, dC, dA, dB, dbias, opts=None):
    """Gradients of :func:`gemm_bias_act` with respect to A, B and bias:

        dZ = dC o act'(Z),  dA = alpha dZ op(B)^T,  dB = alpha op(A)^T dZ,
        dbias = row sums of dZ (column sums where dbias is 1 x n)

    dA and dB have the shapes of op(A) and op(B) (pass a transposed view for an
    operand that entered transposed); None leaves a gradient out.  ``Z`` is what
    the forward pass stored (may be None for the identity).  The residual's
    gradient is beta dC.  dA, dB and dbias overlap no other matrix of the call.
    dZ is rounded to the matrices' type between the two steps, the bias gradient
    is summed from its unrounded values.  With Option.PreciseGradient, what the
    rounding of a 16-bit dZ leaves over enters the products as a second matrix:
    dA and dB are then off by little more than their own rounding (by 1.4 times
    it without), for twice the operations."""
    what, mats = "gemm_bias_act_grad", (A, B, Z, dC, dA, dB, dbias)
    a = _act(act)
    if Z is None and a:
        raise SlateError(f"{what}: Z is wanted for activation {act}")
    with trace_block(what):
        one = _one(mats)
        if one != 1:
            m, n, k = dC.m(), dC.n(), A.n()
            bshape, bmode = _bias_of(what, dbias, m, n)
            _check(dict(A=A, B=B, Z=Z, dC=dC, dA=dA, dB=dB, dbias=dbias),
                   dict(A=(m, k), B=(k, n), Z=(m, n), dC=(m, n), dA=(m, k), dB=(k, n), dbias=bshape), what)
            _apart(what, [("dA", dA), ("dB", dB), ("dbias", dbias)], [("A", A), ("B", B), ("Z", Z), ("dC", dC)],
                   None, not one)
            if not one:
                dZ = _dz_dist(a, dC, (Z if a else None, None), dbias, bmode, _precise(opts, dC.dtype))
                if dA is not None:
                    _run_dist_any(PLAIN, alpha, dZ, [_t(B)] * len(dZ), [dA])
                if dB is not None:
                    _run_dist_any(PLAIN, alpha, [_t(A)] * len(dZ), dZ, [dB])
            if not one or dC.storage.bc.pr < 0:
                return
        oa, ob, oz, oc, ga, gb, gv = _operands(what, ("A", "B", "Z", "dC", "dA", "dB", "dbias"), mats)
        m, n, k = oc.m, oc.n, oa.n
        for name, x, r, c in (("A", oa, m, k), ("B", ob, k, n), ("Z", oz, m, n), ("dA", ga, m, k), ("dB", gb, k, n)):
            _shape(what, name, x, r, c)
        mode = _bias_mode(what, None if dbias is None else (gv.m, gv.n), m, n)
        _outputs(what, (("dA", ga), ("dB", gb), ("dbias", gv)), (("A", oa), ("B", ob), ("Z", oz), ("dC", oc)))
        with _on(oc.t):
            dZ = oc
            if a or mode:
                oz = _NONE if not a else oz if oz.trans == oc.trans else _turn(oz, oc.trans)
                if a and (dA is not None or dB is not None):
                    dZ = None
                if mode and oc.trans:
                    mode = 3 - mode
            if oc.t.is_cuda and m and n:
                made = dZ is None
                two = made and _precise(opts, oc.dt)
                dZ = (oc,) if not made else _DZ[:2] if two else _DZ[:1]
                steps = [oc.rows, oc.cols, a, oc.ptr, oc.ld, oz.ptr, oz.ld, 0, 0, gv.ptr, _inc(gv), mode, made, two, 2]
                tr, how = oc.trans, SUM if two else PLAIN
                _step(steps, how, n if alpha else 0, dZ, tr, (ob,) * len(dZ), not ob.trans, ga)
                _step(steps, how, m if alpha else 0, (oa,) * len(dZ), not oa.trans, dZ, tr, gb)
                _grad_run(alpha, oc, steps)
                _modified(dA, dB, dbias)
                return
            made = dZ is None
            if made:
                dZ = _like(oc, oc.rows, oc.cols, oc.trans)
            parts = [dZ]
            if made and _precise(opts, oc.dt):
                parts.append(_like(oc, oc.rows, oc.cols, oc.trans))
            if a or mode:
                _act_grad(oc.rows, oc.cols, a, oc, oz, _NONE, dZ if made else _NONE, _NONE, gv, mode,
                          rest=(*parts[1:], _NONE, _NONE)[:2])
            if dA is not None:
                _product(PLAIN, alpha, parts, [ob.T] * len(parts), [ga])
            if dB is not None:
                _product(PLAIN, alpha, [oa.T] * len(parts), parts, [gb])
        _modified(dA, dB, dbias)


def _precise(opts, dt):
    """Are the parts of dZ that 16 bits do not hold wanted?"""
    return dt in _HALF and get_option(opts, Option.PreciseGradient, False)


def _product(mode, alpha, A, B, C):
    """One rank's product(s) op(A_i) op(B_i) into outputs of either orientation; those
    of one output are added."""
    if C[0].trans:
        A, B, C = ([x.T for x in y] for y in (B, A, C))
    if mode == PLAIN and len(A) > 1:
        mode = SUM
    (a1, a2), (b1, b2), (c1, c2) = ((*x, _NONE)[:2] for x in (A, B, C))
    _launch(mode, alpha, a1, a2, b1, b2, c1, c2, more=list(zip(A[2:], B[2:])))


def gemm_gated_grad(A1, A2, B, act, Z1, Z2, dC, dA1, dA2, dB, opts=None):
    """Gradients of :func:`gemm_gated`:

        dZ1 = dC o Z2 o act'(Z1),  dZ2 = dC o act(Z1),
        dA1 = dZ1 op(B)^T,  dA2 = dZ2 op(B)^T,  dB = op(A1)^T dZ1 + op(A2)^T dZ2

    with Z1, Z2 as the forward pass stored them; None leaves a gradient out.
    dA1, dA2 and dB overlap no other matrix of the call.
    Both weight gradients are one launch, and dB is one sum over both products,
    rounded once.  dZ1 and dZ2 are rounded to the matrices' type;
    Option.PreciseGradient as for :func:`gemm_bias_act_grad`."""
    what, mats = "gemm_gated_grad", (A1, A2, B, Z1, Z2, dC, dA1, dA2, dB)
    names = ("A1", "A2", "B", "Z1", "Z2", "dC", "dA1", "dA2", "dB")
    a = _act(act)
    if Z1 is None or Z2 is None:
        raise SlateError(f"{what}: Z1 and Z2 are wanted")
    with trace_block(what):
        one = _one(mats)
        if one != 1:
            m, n, k = dC.m(), dC.n(), A1.n()
            w, z = (m, k), (m, n)
            _check(dict(zip(names, mats)), dict(zip(names, (w, w, (k, n), z, z, z, w, w, (k, n)))), what)
            pairs = list(zip(names, mats))
            _apart(what, pairs[6:], pairs[:6], None, not one)
            if not one:
                dZ = _dz_dist(a, dC, (Z1, Z2), None, 0, _precise(opts, dC.dtype))
                for d, g in ((dZ[::2], dA1), (dZ[1::2], dA2)):
                    if g is not None:
                        _run_dist_any(PLAIN, 1.0, d, [_t(B)] * len(d), [g])
                if dB is not None:
                    _run_dist_any(SUM, 1.0, [_t(A1), _t(A2)] * (len(dZ) // 2), dZ, [dB])
            if not one or dC.storage.bc.pr < 0:
                return
        o1, o2, ob, z1, z2, oc, g1, g2, gb = opds = _operands(what, names, mats)
        m, n, k = oc.m, oc.n, o1.n
        w, z = (m, k), (m, n)
        for name, x, (r, c) in zip(names, opds, (w, w, (k, n), z, z, z, w, w, (k, n))):
            _shape(what, name, x, r, c)
        pairs = tuple(zip(names, opds))
        _outputs(what, pairs[6:], pairs[:6])
        with _on(oc.t):
            tr = oc.trans
            if z1.trans != tr:
                z1 = _turn(z1, tr)
            if z2.trans != tr:
                z2 = _turn(z2, tr)
            if dB is not None and o2.trans != o1.trans:
                o2 = _turn(o2, o1.trans)
            if oc.t.is_cuda and m and n:
                two = _precise(opts, oc.dt)
                steps = [oc.rows, oc.cols, a, oc.ptr, oc.ld, z1.ptr, z1.ld, z2.ptr, z2.ld, 0, 1, 0, 2, two, 4 if two else 2]
                if two:
                    _step(steps, SUM, n, _DZ[::2], tr, (ob, ob), not ob.trans, g1)
                    _step(steps, SUM, n, _DZ[1::2], tr, (ob, ob), not ob.trans, g2)
                elif dA1 is not None and dA2 is not None and g1.trans == g2.trans:
                    _step(steps, PAIR, n, _DZ[:2], tr, (ob, ob), not ob.trans, g1, g2)
                else:
                    _step(steps, PLAIN, n, _DZ[:1], tr, (ob,), not ob.trans, g1)
                    _step(steps, PLAIN, n, _DZ[1:2], tr, (ob,), not ob.trans, g2)
                _step(steps, SUM, m, (o1, o2, o1, o2) if two else (o1, o2), not o1.trans, _DZ if two else _DZ[:2], tr, gb)
                _grad_run(1.0, oc, steps)
                _modified(dA1, dA2, dB)
                return
            d = [_like(oc, oc.rows, oc.cols, tr) for _ in range(4 if _precise(opts, oc.dt) else 2)]
            _act_grad(oc.rows, oc.cols, a, oc, z1, z2, d[0], d[1], rest=(*d[2:], _NONE, _NONE)[:2])
            if dA1 is not None and dA2 is not None and g1.trans == g2.trans and len(d) == 2:
                _product(PAIR, 1.0, d, [ob.T, ob.T], [g1, g2])
            else:
                for x, g in ((d[::2], g1), (d[1::2], g2)):
                    if g.t is not None:
                        _product(PLAIN, 1.0, x, [ob.T] * len(x), [g])
            if dB is not None:
                _product(SUM, 1.0, [o1.T, o2.T] * (len(d) // 2), d, [gb])
        _modified(dA1, dA2, dB)


def _run_dist_any(mode, alpha, A, B, C):
    """_run_dist into outputs of either orientation; products of one output are added."""
    if mode == PLAIN and len(A) > 1:
        mode = SUM
    if C[0]._op != Op.NoTrans:
        A, B, C = [_t(x) for x in B], [_t(x) for x in A], [_t(x) for x in C]
    _run_dist(mode, alpha, A, B, C)


def _dz_dist(act, dC, Z, dbias, bmode, precise):
    """dZ (one or two matrices, from offset 0 on dC's grid; precise: behind them
    what their rounding leaves over) and the bias gradient: local sums in 32 (64) bits, one all-reduce over the process row
    (column), one rounding."""
    W = dC if dC.storage.bc.mb == dC.storage.bc.nb and _placed(dC, dC) else None
    if W is None:
        W = _grid_work(dC, dC.m(), dC.n())
        from ..parallel.redist import redistribute_pieces
        redistribute_pieces(dC, W)
    Zw = [None if z is None else _onto(z, W) for z in Z]
    two = Zw[1] is not None
    made = 2 if two else 1
    dZ = [_grid_work(W, dC.m(), dC.n()) for _ in range(2 * made if precise else made)] if act or two else [W]
    lb, s = W.local_block(), W.storage
    db, sums = _NONE, None
    if dbias is not None:
        wide = torch.float64 if s.dtype == torch.float64 else torch.float32
        sums = torch.zeros(lb.mloc if bmode == 1 else lb.nloc, dtype=wide, device=lb.data.device)
        db = _Opd(sums.data_ptr(), sums.numel(), sums.numel(), 1, False, sums.view(-1, 1))
    if s.bc.pr >= 0 and (act or two or dbias is not None):
        oz = [_NONE if z is None else _opd(z) for z in Zw]
        od = [_opd(d) for d in dZ] if act or two else [_NONE]
        with _on(lb.data):
            _act_grad(lb.mloc, lb.nloc, act, _opd(W), oz[0], oz[1], od[0], od[1] if two else _NONE, db, bmode, True,
                      (*od[made:], _NONE, _NONE)[:2])
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
    """Operands of a list of matrices of one type, device and communicator, and
    the storages among theirs whose state a write changes."""
    if not isinstance(mats, (list, tuple)):
        raise SlateError(f"{what}: a list of matrices is wanted")
    out, todo, dt, dev, comm = [], [], None, None, None
    add, anew = out.append, debug_checks()
    for M in mats:
        s = M.storage
        slot, table = s.origin_slot, s.table
        x = M.__dict__.get("_operand")
        # (the use of a remembered operand, as in _opd, without the call)
        now = table.version()
        if not M._whole or x is None or x.version != now or x.table is not table or x.t.data_ptr() != x.ptr or anew:
            if not M._whole or s.bc is None:
                raise SlateError(f"{what}: general block-cyclic matrices are wanted")
            if slot is None:
                raise SlateError(f"{what}: a matrix has no tiles (insertLocalTiles)")
            x = _opd(M)
            now = table.version()
        if dt is None:
            dt, dev, comm = x.dt, x.dev, s.comm
        elif x.dt is not dt or x.dev is not dev:
            raise SlateError(f"{what}: the matrices differ in type or device ({x.dt} on {x.dev}, {dt} on {dev})")
        elif s.comm is not comm and s.comm.ranks != comm.ranks:
            raise SlateError(f"{what}: the matrices differ in communicator")
        if anew or s._marked != (slot, now):
            todo.append(s)
        add(x)
    return out, todo


def _clip_apart(what, va, vb):
    """What is written shares no element with another matrix of the call."""
    todo = [(y.ptr, y.end, i) for i, y in enumerate(vb)]
    if vb is not va:
        todo += [(x.ptr, x.end, ~i) for i, x in enumerate(va)]
    todo.sort()
    last = 0
    for lo, hi, _ in todo:
        if lo < last and hi > lo:
            break
        last = max(last, hi)
    else:
        return
    # address ranges overlap: element by element, each against those that begin inside it
    for i, (_, hi, p) in enumerate(todo):
        x = vb[p] if p >= 0 else va[~p]
        for lo, _, q in todo[i + 1:]:
            if lo >= hi:
                break
            y = vb[q] if q >= 0 else va[~q]
            if y.end == y.ptr or p < 0 and q < 0 or p == ~q and (x.ptr, x.ld, x.dt) == (y.ptr, y.ld, y.dt):
                continue
            if _overlap(x, y):
                raise SlateError(f"{what}: matrices {p if p >= 0 else ~p} and {q if q >= 0 else ~q} of the call overlap")


def _clip_apart_grid(what, A, B, va, vb):
    """:func:`_clip_apart` on a grid of ranks.  Views of one storage are compared
    by their global indexes, and refused on every rank alike; -> what buffers of
    the caller share on this rank."""
    views = {}
    for i, M in enumerate(B):
        views.setdefault(id(M.storage), []).append((i, True, M))
    if B is not A:
        for i, M in enumerate(A):
            views.setdefault(id(M.storage), []).append((i, False, M))
    for group in views.values():
        for k, (i, w, X) in enumerate(group):
            for j, v, Y in group[:k]:
                if (w or v) and _share(X, Y, i == j and w is not v):
                    raise SlateError(f"{what}: matrices {j} and {i} of the call overlap")
    if len(views) > 1 and any(M.storage.wraps for M in (*A, *B)):
        try:
            _clip_apart(what, va, vb)
        except SlateError as e:
            return e
    return None


def clip_norm(max_norm, A, B=None, opts=None):
    """B_i = min(1, max_norm / s) A_i with s the Frobenius norm of all matrices
    of the list A together; returns s as a float64 tensor on the matrices'
    device (no host synchronisation).

    B = None scales in place.  B's matrices have A's shapes and distribution,
    and A's type or, for 16-bit A, float32.  Where s is not finite the matrices
    are copied (left) as they are, so that a caller can look at s and skip the
    step.  The squares are summed in 64 bits, in an order that depends on the
    sizes alone.  Matrices written overlap no other matrix of the call, except
    that B_i may be A_i.  (On a grid, where buffers of the caller do so on some
    ranks only, those ranks raise and s is NaN on the others.)"""
    what = "clip_norm"
    limit = float(max_norm)
    if not limit >= 0:
        raise SlateError(f"{what}: max_norm {max_norm} is not >= 0")
    return _clip(what, limit, A, A if B is None else B)


def global_norm(A, opts=None):
    """Frobenius norm of all matrices of the list A together (a float: waits
    for the device, as ``norm`` does)."""
    return float(_clip("global_norm", None, A, A))


_PARTS = {torch.complex64: torch.float32, torch.complex128: torch.float64}


def _clip(what, limit, A, B):
    va, todo = _clip_views(A, what)
    if not va:
        return torch.zeros((), dtype=torch.float64)
    vb = va
    if B is not A:
        vb, todo = _clip_views(B, what)
    t, comm = va[0].t, A[0].storage.comm
    if len(vb) != len(va) or (vb is not va and vb[0].dev is not va[0].dev):
        raise SlateError(f"{what}: B has {len(vb)} matrices, A has {len(va)}, or they are on different devices")
    ta, tb = va[0].dt, vb[0].dt
    if _PARTS.get(ta, ta) not in REAL_CODE or not (ta == tb or (_BYTES[ta] == 2 and tb == torch.float32)):
        raise SlateError(f"{what}: no scaling from {ta} to {tb}")
    two = 2 if ta in _PARTS else 1
    ca, cb = REAL_CODE[_PARTS.get(ta, ta)], REAL_CODE[_PARTS.get(tb, tb)]
    with trace_block(what):
        # (A, lda, B, ldb, rows, columns) of every matrix; complex ones as pairs
        mats = []
        for x, y in zip(va, vb):
            rows, cols = x.rows, x.cols
            if rows != y.rows or cols != y.cols or x.trans is not y.trans:
                raise SlateError(f"{what}: B's matrices want the shapes and ops of A's")
            mats += (x.ptr, x.ld * two, y.ptr, y.ld * two, rows * two, cols)
        if vb is not va and comm.size > 1:
            for X, Y in zip(A, B):
                if X.m() != Y.m() or X.n() != Y.n() or not _same_place(X, Y):
                    raise SlateError(f"{what}: B's matrices want the shapes and distribution of A's")
        mod, st = kmod(t), raw_stream(t)
        top, scale = (0.0, False) if limit is None else (limit, True)
        with _on(t):
            # [norm, the ranks' common sums (3), partial sums]
            ws = torch.empty(4 + mod.clip_parts(len(va)), dtype=torch.float64, device=t.device)
            norm = ws.data_ptr()
            part = norm + 32
            if comm.size == 1:
                if not mod.clip_norm(ca, cb, mats, top, part, norm, scale, True, st):
                    _clip_apart(what, va, vb)
                    mod.clip_norm(ca, cb, mats, top, part, norm, scale, False, st)
            else:
                shared = _clip_apart_grid(what, A, B, va, vb) if scale else None
                n = mod.clip_sum(ca, mats, part, st)
                mod.clip_join(part, n, norm + 8, st)
                if shared is not None:
                    # the others are in the sum already: a NaN keeps them from scaling
                    ws[1:4].fill_(float("nan"))
                comm.allreduce(ws[1:4], "sum")
                if shared is not None:
                    raise shared
                mod.clip_scale(ca, cb, mats, top, norm + 8, 1, norm, scale, st)
        if scale:
            for s in todo:
                s.mark_local_modified(s.origin_slot)
    return ws[0]


def _same_place(X, Y):
    """The same tiles of the same grid, from the same offset (the shapes may differ)."""
    a, b = X.storage.bc, Y.storage.bc
    return (a.mb, a.nb, a.p, a.q, a.order) == (b.mb, b.nb, b.p, b.q, b.order) and \
        X.global_offsets() == Y.global_offsets() and X.storage.comm.ranks == Y.storage.comm.ranks

"""Helpers of the tests of the seam's operators: bf16 as uint16 arrays, padded
matrices in device memory, and the calls on them."""
import ctypes

import numpy as np

from macboost_amd import _core

HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8}      # half a step of rounding, relative


def to_bf16(a):
    """float32 -> bf16 bits, to nearest even."""
    b = np.ascontiguousarray(a, np.float32).view(np.uint32)
    r = (b + 0x7FFF + ((b >> 16) & 1)) >> 16
    return np.where(np.isnan(a), 0x7FC0, r).astype(np.uint16)


def from_bf16(b):
    return (np.asarray(b, np.uint16).astype(np.uint32) << 16).view(np.float32)


def encode(a, kind):
    return to_bf16(a) if kind == "bf16" else np.ascontiguousarray(a, np.float32)


def decode(a, kind):
    return from_bf16(a) if kind == "bf16" else a


def rounded(a, kind):
    """The values of `a` that a matrix of that type holds."""
    return decode(encode(a, kind), kind).reshape(np.shape(a))


def padded(a, kind, pad, fill):
    """[rows][cols + pad] of the type, `fill` between the rows."""
    full = np.full((a.shape[0], a.shape[1] + pad), fill, np.float32)
    full[:, :a.shape[1]] = a
    return encode(full, kind)


def ptr(p):
    return None if p is None else ctypes.c_void_p(p)


class Xent:
    """One problem of the many-class loss in device memory."""

    def __init__(self, ctx, h, w, labels, kind, bias=None, weights=None, h_pad=0, w_pad=0,
                 guard=7.0):
        self.ctx, self.kind, self.guard = ctx, kind, guard
        self.n, self.d = h.shape
        self.v = w.shape[0]
        self.h_pad, self.w_pad = h_pad, w_pad
        up = ctx.upload
        self.h = up(padded(h, kind, h_pad, np.nan))
        self.w = up(padded(w, kind, w_pad, np.nan))
        self.labels = up(np.asarray(labels, np.int32))
        self.bias = None if bias is None else up(np.asarray(bias, np.float32))
        self.weights = None if weights is None else up(np.asarray(weights, np.float32))
        self.loss = up(np.full(max(1, self.n), guard, np.float32))
        self.lse = up(np.full(max(1, self.n), guard, np.float32))
        self.dh = up(padded(np.full(h.shape, guard), kind, h_pad, guard))
        self.dw = up(padded(np.full(w.shape, guard), kind, w_pad, guard))
        self.db = up(np.full(self.v, guard, np.float32))
        self.shape = _core.MbkXentShape(self.n, self.v, self.d,
                                        _core.BF16 if kind == "bf16" else _core.F32,
                                        self.d + h_pad, self.d + w_pad)

    def forward(self):
        self.ctx.call("mbk_xent", ctypes.byref(self.shape), self.h, self.w, ptr(self.bias),
                      self.labels, ptr(self.weights), self.loss, self.lse)

    def grad(self, dh=True, dw=True, db=True):
        self.ctx.call("mbk_xent_grad", ctypes.byref(self.shape), self.h, self.w, ptr(self.bias),
                      self.labels, ptr(self.weights), self.loss, self.lse,
                      self.dh if dh else None, self.dw if dw else None, self.db if db else None)

    def _matrix(self, p, rows, pad):
        dtype = np.uint16 if self.kind == "bf16" else np.float32
        full = decode(self.ctx.download(p, (rows, self.d + pad), dtype), self.kind)
        assert np.all(full[:, self.d:] == self.guard), "written between the rows"
        return full[:, :self.d]

    def results(self, grad=True):
        self.ctx.sync()
        out = {"loss": self.ctx.download(self.loss, self.n, np.float32),
               "lse": self.ctx.download(self.lse, self.n, np.float32)}
        if grad:
            out["dh"] = self._matrix(self.dh, self.n, self.h_pad)
            out["dw"] = self._matrix(self.dw, self.v, self.w_pad)
            out["db"] = self.ctx.download(self.db, self.v, np.float32)
        return out


def xent_reference(h, w, labels, kind, bias=None, weights=None):
    """The loss and its gradients in 64 bits, and how far each may be off.

    Half a step of the operands' splitting (f32: two f16 terms hold 22 bits, and what the
    three products drop is as much again; bf16: one term holds it, G has 11 bits) and of
    f32 sums of as many terms as there are is carried through the formulas, worst case
    in every term."""
    h, w = rounded(h, kind).astype(np.float64), rounded(w, kind).astype(np.float64)
    n, d = h.shape
    v = w.shape[0]
    b = np.zeros(v) if bias is None else np.asarray(bias, np.float32).astype(np.float64)
    wt = np.ones(n) if weights is None else np.asarray(weights, np.float32).astype(np.float64)
    labels = np.asarray(labels)
    closed = b == -np.inf
    w = np.where(closed[:, None], 0.0, w)
    live = (labels >= 0) & (labels < v) & (wt != 0) & (not closed.all())
    u = 2.0 ** -24
    split = 0.0 if kind == "bf16" else 3 * 2.0 ** -22
    products = 1 if kind == "bf16" else 3
    with np.errstate(all="ignore"):
        z = np.where(closed, -np.inf, h @ w.T + b)
        size = np.abs(h) @ np.abs(w).T
        ez = size * (split + (products * d + 16) * u) + np.where(closed, 0, np.abs(z)) * 2 * u \
            + np.where(closed, 0, np.abs(b)) * u
        top = z.max(1)
        ref = np.where(np.isfinite(top), top, 0)
        p = np.exp(z - ref[:, None])
        lse = ref + np.log(p.sum(1))
        off = np.where(closed, 0, ez).max(1)
        elz = off + (v + 32) * u + 4 * u * np.maximum(1, np.abs(lse))
        out = {"lse": (lse, elz)}
        hl = np.where(live[:, None], h, 0.0)
        at = np.where(live, labels, 0)
        zy = z[np.arange(n), at]
        wl = np.where(live, wt, 0.0)
        loss = np.where(live, wt * (lse - zy), 0.0)
        out["loss"] = (loss, np.abs(wl) * (elz + np.where(live, ez[np.arange(n), at], 0)
                                           + 2 * u * np.where(live, np.abs(lse - zy), 0)))
        p = np.exp(z - np.where(np.isfinite(lse), lse, 0)[:, None])
        p[~live] = 0
        hot = np.zeros((n, v))
        hot[np.arange(n)[live], labels[live]] = 1
        g = (p - hot) * wl[:, None]
        # the exponent's and exp2's own errors, and G's rounding
        dist = np.where(closed, 0, np.abs(z - lse[:, None]))
        rel = np.where(closed, 0, ez) + elz[:, None] + (3 * dist + 8) * u
        half = 2.0 ** -11 if kind == "bf16" else 2.0 ** -22     # G in one f16 term or two
        eg = np.abs(wl)[:, None] * (p * rel + np.abs(p - hot) * half + 2.0 ** -38)
        # f16 terms of G times the row's weight share one scale, that of the largest row
        rows = np.abs(hl).max(1) if d else np.zeros(n)
        with_scale = 2.0 ** -37 * (np.abs(wl) * rows).max(initial=0)
        ew = eg + np.where(rows > 0, with_scale / np.where(rows > 0, rows, 1), 0)[:, None]
        for e in (eg, ew, g):
            e[~live] = 0
            e[:, closed] = 0

        def product(left, right, e_left, e_right, terms):
            return (e_left @ np.abs(right) + np.abs(left) @ e_right
                    + (np.abs(left) @ np.abs(right)) * (split + (products * terms + 16) * u))

        # bf16: the row's weight goes into h's f16 term, or into G's
        none_w, off_h = np.zeros_like(w), np.abs(hl) * (2.0 ** -11 if kind == "bf16" else 0.0)
        for name, value, err in (
                ("dh", g @ w, product(g, w, eg, none_w, v)),
                ("dw", g.T @ hl, product(g.T, hl, ew.T, off_h, n)),
                ("db", g.sum(0), eg.sum(0) + np.abs(g).sum(0) * (n + 4) * u)):
            step = HALF[kind] if name != "db" else u
            out[name] = (value, err + (np.abs(value) + err) * step + 1e-37)
    return out


def check(got, want, names=("loss", "lse", "dh", "dw", "db")):
    for name in names:
        value, tol = want[name]
        a = got[name].astype(np.float64)
        same = (a == value) | (np.isnan(a) & np.isnan(value))
        bad = ~same & ~(np.abs(a - value) <= tol)
        assert not bad.any(), (name, np.argwhere(bad)[:3], a[bad][:3], value[bad][:3], tol[bad][:3])


class Experts:
    """A sort by expert in device memory."""

    def __init__(self, ctx, expert, experts):
        self.ctx = ctx
        self.rows, self.k = expert.shape
        self.experts = experts
        n = max(1, expert.size)
        self.expert = ctx.upload(expert.astype(np.int32) if expert.size else np.zeros(1, np.int32))
        self.offsets = ctx.upload(np.full(experts + 1, -7, np.int32))
        self.source = ctx.upload(np.full(n, -7, np.int32))
        self.slot = ctx.upload(np.full(n, -7, np.int32))
        self.plan = _core.MbkExpertPlan(self.rows, self.k, experts, self.expert, self.offsets,
                                        self.source, self.slot)

    def sort(self):
        self.ctx.call("mbk_expert_sort", ctypes.byref(self.plan))

    def order(self):
        self.ctx.sync()
        n = self.rows * self.k
        return (self.ctx.download(self.offsets, self.experts + 1, np.int32),
                self.ctx.download(self.source, n, np.int32),
                self.ctx.download(self.slot, (self.rows, self.k), np.int32))


def sort_reference(expert, experts):
    flat = expert.ravel()
    kept = np.flatnonzero((flat >= 0) & (flat < experts))
    order = kept[np.argsort(flat[kept], kind="stable")]
    source = np.full(flat.size, -1, np.int64)
    source[:order.size] = order
    slot = np.full(flat.size, -1, np.int64)
    slot[order] = np.arange(order.size)
    offsets = np.concatenate([[0], np.cumsum(np.bincount(flat[kept], minlength=experts))])
    return offsets, source, slot.reshape(expert.shape)


def to_sorted(rows, offsets, blocked):
    """[slots][cols] as the sorted matrix lies in memory."""
    if not blocked:
        return rows.ravel().copy()
    out = rows.ravel().copy()
    cols = rows.shape[1]
    for a, b in zip(offsets[:-1], offsets[1:]):
        out[a * cols:b * cols] = rows[a:b].T.ravel()
    return out


def from_sorted(flat, offsets, cols, blocked):
    out = flat.reshape(-1, cols).copy()
    if blocked:
        for a, b in zip(offsets[:-1], offsets[1:]):
            out[a:b] = flat[a * cols:b * cols].reshape(cols, b - a).T
    return out


def rows_matrix(ctx, a, kind, major, pad, blocked, fill=np.nan):
    """`a` [rows][cols] in device memory, rows or columns padded: (pointer, structure)."""
    m = a if major == "row" else a.T
    p = ctx.upload(padded(m, kind, pad, fill))
    stride = m.shape[1] + pad
    row, col = (stride, 1) if major == "row" else (1, stride)
    return p, _core.MbkExpertMatrix(p, row, col, a.shape[1],
                                    _core.BF16 if kind == "bf16" else _core.F32, int(blocked))


def read_rows(ctx, p, rows, cols, kind, major, pad, fill):
    shape = (rows, cols) if major == "row" else (cols, rows)
    dtype = np.uint16 if kind == "bf16" else np.float32
    full = decode(ctx.download(p, (shape[0], shape[1] + pad), dtype), kind)
    assert np.all(full[:, shape[1]:] == fill), "written between the rows"
    m = full[:, :shape[1]]
    return m if major == "row" else m.T

"""Helpers of the tests of category vectors, clipped gradients, scores from class vectors in 4
bits and their penalties: the calls on padded matrices in device memory, and the same in 64 bits
with how far each result may be off (half steps of rounding, carried through the formulas)."""
import ctypes

import numpy as np

import device_ops as D
from macboost_amd import _core

U = 2.0 ** -24
GUARD = 7.0
CODE = {"f32": _core.F32, "bf16": _core.BF16}
SIZE = {"f32": 4, "bf16": 2}
DTYPE = {"f32": np.float32, "bf16": np.uint16}


def close(got, want, tol):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    same = (got == want) | (np.isnan(got) & np.isnan(want))
    with np.errstate(invalid="ignore"):
        bad = ~same & ~(np.abs(got - want) <= tol)
    tol = np.broadcast_to(tol, want.shape)
    assert not bad.any(), (np.argwhere(bad)[:3], got[bad][:3], want[bad][:3], tol[bad][:3],
                           int(bad.sum()))


class Matrix:
    """[rows][cols] of the type in device memory, pad elements of GUARD (or `fill`) behind each
    row, and `shift` elements before the first."""

    def __init__(self, ctx, a, kind, pad=0, shift=0, fill=GUARD):
        self.ctx, self.kind, self.pad, self.shift, self.fill = ctx, kind, pad, shift, fill
        self.rows, self.cols = a.shape
        self.stride = self.cols + pad
        full = np.full(shift + self.rows * self.stride + 1, fill, np.float32)
        full[shift:shift + self.rows * self.stride].reshape(
            self.rows, self.stride)[:, :self.cols] = a
        self.at = ctx.upload(D.encode(full, kind))
        self.ptr = self.at + shift * SIZE[kind]

    def read(self):
        n = self.shift + self.rows * self.stride + 1
        full = D.decode(self.ctx.download(self.at, n, DTYPE[self.kind]), self.kind)
        body = full[self.shift:-1].reshape(self.rows, self.stride)
        assert np.all(full[:self.shift] == self.fill) and full[-1] == self.fill
        assert np.all(body[:, self.cols:] == self.fill), "written between the rows"
        return body[:, :self.cols]


def blank(ctx, rows, cols, kind, pad=0, shift=0):
    return Matrix(ctx, np.full((rows, cols), GUARD, np.float32), kind, pad, shift)


def embed_shape(rows, entries, dim, kind, row_stride, table_stride, scale=1.0):
    return ctypes.byref(_core.MbkEmbedShape(rows, entries, dim, CODE[kind], row_stride,
                                            table_stride, scale))


def embed_reference(table, ids, base, scale, kind):
    entries = table.shape[0]
    kept = (ids >= 0) & (ids < entries)
    v = np.where(kept[:, None], table[np.where(kept, ids, 0)].astype(np.float64), 0.0)
    out = np.float64(np.float32(scale)) * v + (0.0 if base is None else base.astype(np.float64))
    return out, np.abs(out) * (U + D.HALF[kind]) * (1 + U) + 1e-44


def embed_grad_reference(dout, ids, entries, base, scale, kind):
    kept = np.flatnonzero((ids >= 0) & (ids < entries))
    order = kept[np.argsort(ids[kept], kind="stable")]
    total = np.zeros((entries, dout.shape[1]))
    size, terms = np.zeros_like(total), np.zeros((entries, 1))
    if order.size:
        used, first = np.unique(ids[order], return_index=True)
        rows = dout[order].astype(np.float64)
        total[used] = np.add.reduceat(rows, first, axis=0)
        size[used] = np.add.reduceat(np.abs(rows), first, axis=0)
        terms[used, 0] = np.diff(np.append(first, order.size))
    by = np.float64(np.float32(scale))
    out = total * by + (0.0 if base is None else base.astype(np.float64))
    # at most terms - 1 additions whatever their order, and the sum with base
    off = size * terms * U * abs(by)
    return out, off + (np.abs(out) + off) * (U + D.HALF[kind]) * (1 + U) + 1e-44


def quantised(w, group):
    """Codes and scales of W, [classes][groups * group] and [classes][groups]."""
    v, d = w.shape
    groups = -(-d // group)
    full = np.zeros((v, groups * group), np.float32)
    full[:, :d] = w
    full = full.reshape(v, groups, group)
    scale = D.rounded(np.abs(full).max(2) * np.float32(1 / 7), "bf16").astype(np.float32)
    with np.errstate(all="ignore"):
        code = np.where(scale[:, :, None] > 0, np.rint(full / scale[:, :, None]), 0)
    return np.clip(code, -8, 7).astype(np.int8).reshape(v, -1), scale


def values(code, scale, dim):
    v, groups = scale.shape
    return (code.reshape(v, groups, -1).astype(np.float64)
            * scale[:, :, None].astype(np.float64)).reshape(v, -1)[:, :dim]


class Fourbit:
    """W in 4 bits in device memory."""

    def __init__(self, ctx, w, kind, group, pad=0):
        self.ctx, self.kind = ctx, kind
        self.classes, self.dim = w.shape
        self.group = group
        self.shape = _core.MbkFourbitShape(self.classes, self.dim, group)
        self.bytes = _core.fourbit_bytes(self.shape)
        w = Matrix(ctx, w, kind, pad, fill=np.nan)
        self.packed = ctx.upload(np.full(self.bytes + 64, 0xA5, np.uint8))
        ctx.call("mbk_fourbit_pack", ctypes.byref(self.shape), CODE[kind], w.ptr, w.stride,
                 self.packed)
        ctx.sync()

    def read(self):
        """The codes and scales that the packed form holds, by its layout."""
        raw = self.ctx.download(self.packed, self.bytes + 64, np.uint8)
        assert np.all(raw[self.bytes:] == 0xA5), "written behind the packed form"
        tiles, blocks, per = -(-self.classes // 16), -(-self.dim // 128), 128 // self.group
        words = raw[:tiles * blocks * 1024].view(np.uint32).reshape(tiles, blocks, 4, 16, 4)
        code = np.zeros((tiles, blocks, 4, 16, 4, 8), np.int8)     # tile, block, q, class, j, i
        for i in range(8):
            code[..., i] = ((words >> (4 * ((i >> 1) + 4 * (i & 1)))) & 15).astype(np.int8) - 8
        # element 32 j + 8 q + i
        code = code.transpose(0, 3, 1, 4, 2, 5).reshape(tiles * 16, blocks * 128)
        at = tiles * blocks * 1024
        quads = -(-blocks // 4)
        size = tiles * quads * 16 * 4 * per * 2
        half = raw[at:at + size].view(np.float16).reshape(tiles, quads, 16, 4 * per)
        at += -(-size // 256) * 256
        exponent = raw[at:at + tiles * 64].view(np.int32)
        scale = half.astype(np.float64).transpose(0, 2, 1, 3).reshape(tiles * 16, quads * 4 * per)
        return code, np.ldexp(scale, exponent[:, None])

    def scores(self, h, bias=None, pad=0, score_pad=0, shift=0, out=None):
        rows = h.shape[0]
        hm = Matrix(self.ctx, h, self.kind, pad, shift, fill=np.nan)
        out = blank(self.ctx, rows, self.classes, "f32", score_pad) if out is None else out
        b = None if bias is None else self.ctx.upload(np.asarray(bias, np.float32))
        self.ctx.call("mbk_fourbit_scores", ctypes.byref(self.shape), rows, CODE[self.kind], hm.ptr,
                      hm.stride, self.packed, b, out.ptr, out.stride)
        self.ctx.sync()
        return out.read()


def scores_reference(h, w, bias, kind):
    """h . w + bias in 64 bits of what the types hold, and how far off: a step for each of the
    f32 additions, the half steps of two f16 terms of f32 h (22 bits), the bias and its sum."""
    h = h.astype(np.float64)
    z = h @ w.T
    size = np.abs(h) @ np.abs(w).T
    terms = 2 if kind == "f32" else 1
    off = size * ((terms * (h.shape[1] + 127) + 16) * U + (2.0 ** -22 if kind == "f32" else 0.0))
    # what is small beside the row's largest |h|, or the class's largest |w|
    off = off + np.abs(h).max(1)[:, None] * 2.0 ** -38 * np.abs(w).sum(1)[None] + \
        np.abs(w).max(1)[None] * 2.0 ** -36 * np.abs(h).sum(1)[:, None]
    off = off + np.abs(z) * U
    if bias is None:
        return z, off + 1e-44
    b = np.asarray(bias, np.float32).astype(np.float64)
    out = np.where(b == -np.inf, -np.inf, z + np.where(b == -np.inf, 0, b))
    return out, off + np.where(b == -np.inf, 0, np.abs(z + np.where(b == -np.inf, 0, b))) * U + 1e-44


def adjust_reference(scores, ids, lengths, bias, allowed, repetition, presence, frequency):
    n, v = scores.shape
    rep, pres, freq = (np.float64(np.float32(x)) for x in (repetition, presence, frequency))
    z = scores.astype(np.float64)
    off = np.zeros_like(z)
    for r in range(n):
        h = ids[r] if lengths is None else ids[r, :min(max(lengths[r], 0), ids.shape[1])]
        h = h[(h >= 0) & (h < v)]
        at, count = np.unique(h, return_counts=True)
        was = z[r, at]
        with np.errstate(invalid="ignore"):
            by = np.where(was > 0, was / rep, was * rep)
            pen = pres + freq * count
            z[r, at] = by - pen
            off[r, at] = (np.abs(by) + np.abs(pen) + np.abs(by - pen)) * U
    if bias is not None:
        z = z + np.asarray(bias, np.float64)
        off = off + np.abs(z) * U
    if allowed is not None:
        words = np.broadcast_to(allowed, (n, allowed.shape[1])).copy()
        on = np.unpackbits(words.view(np.uint8), axis=1, bitorder="little")[:, :v].astype(bool)
        z = np.where(on, z, -np.inf)
    off = np.where(np.isfinite(off), off, 0)
    return z, off * (1 + 4 * U) + 1e-44

"""Outputs of more than 32 MB, which are stored past the caches: category vectors, their gradient,
clipped gradients and penalties, with values of their own in each row and column."""
import numpy as np
import pytest

import device_ops as D
import macboost_amd as mb
import model_ops as M
from test_gpu_adjust import _adjust, _case
from test_gpu_category_exact import _whole
from test_gpu_category_vectors import _ids
from test_gpu_clip import _clip, _entry, _make, _norm

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = mb.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("kind,rows,dim,pad", [("f32", 140000, 70, 1), ("bf16", 250000, 77, 2),
                                               ("bf16", 270001, 64, 0), ("f32", 2900000, 3, 0)])
def test_lookup(ctx, kind, rows, dim, pad):
    rng = np.random.default_rng(rows)
    entries = 20000
    ids = _ids(rng, rows, entries)
    table, base = _whole(rng, entries, dim, 100), _whole(rng, rows, dim, 100)
    kept = (ids >= 0) & (ids < entries)
    found = np.where(kept[:, None], table[np.where(kept, ids, 0)], np.float32(0)) * np.float32(0.5)
    t, idev = M.Matrix(ctx, table, kind, pad, fill=np.nan), ctx.upload(ids)
    shape = M.embed_shape(rows, entries, dim, kind, dim + pad, t.stride, 0.5)
    for of in (None, base):
        want = D.rounded(found if of is None else found + of, kind)
        b = None if of is None else M.Matrix(ctx, of, kind, pad, fill=np.nan)
        out = M.blank(ctx, rows, dim, kind, pad)
        ctx.call("mbk_embed", shape, t.ptr, idev, None if b is None else b.ptr, out.ptr)
        ctx.sync()
        assert np.array_equal(out.read(), want)
    out = M.Matrix(ctx, base, kind, pad)                 # in place
    ctx.call("mbk_embed", shape, t.ptr, idev, out.ptr, out.ptr)
    ctx.sync()
    assert np.array_equal(out.read(), want)


@pytest.mark.parametrize("kind,rows,dim,entries,pad", [
    # one launch, and a sorted list; last pieces of 16 bytes that share columns
    ("f32", 1000, 70, 140000, 1), ("bf16", 1000, 77, 250000, 0), ("f32", 50000, 70, 140000, 0),
    ("bf16", 50000, 77, 250000, 3), ("f32", 20000, 301, 30000, 0), ("bf16", 100000, 1025, 17000, 1),
    # narrow rows, which stay in the caches
    ("f32", 40000, 3, 3000000, 0),
])
def test_gradient(ctx, kind, rows, dim, entries, pad):
    rng = np.random.default_rng(entries)
    ids = _ids(rng, rows, entries, 1.0)
    kept = (ids >= 0) & (ids < entries)
    dout = _whole(rng, rows, dim, 4)
    assert np.bincount(ids[kept]).max() * 4 < 2 ** 22    # sums that f32 holds, and their halves
    total = np.stack([np.bincount(ids[kept], dout[kept, c], entries) for c in range(dim)], 1)
    idev, g = ctx.upload(ids), M.Matrix(ctx, dout, kind, pad, fill=np.nan)
    shape = M.embed_shape(rows, entries, dim, kind, g.stride, dim + pad, 0.5)
    base = _whole(rng, entries, dim, 8)
    for of in (None, base):
        b = None if of is None else M.Matrix(ctx, of, kind, pad, fill=np.nan)
        want = (total * 0.5 + (0.0 if of is None else of)).astype(np.float32)
        out = M.blank(ctx, entries, dim, kind, pad)
        ctx.call("mbk_embed_grad", shape, idev, g.ptr, None if b is None else b.ptr, out.ptr)
        ctx.sync()
        assert np.array_equal(out.read(), D.rounded(want, kind))


@pytest.mark.parametrize("n,v,hist,pad", [(100, 90001, 300, 3), (130, 65536, 40, 0), (90000, 101, 9, 2)])
def test_penalties(ctx, n, v, hist, pad):
    _, scores, ids, lengths, bias, allowed = _case(n + v, n, v, hist)
    got = _adjust(ctx, scores, ids, lengths, bias, allowed, 1.3, 0.2, 0.1, pad=pad, out_pad=pad + 2,
                  shift=pad % 2, mask_pad=1)
    M.close(got, *M.adjust_reference(scores, ids, lengths, bias, allowed, 1.3, 0.2, 0.1))
    got = _adjust(ctx, scores, ids, None, None, allowed[:1], 0.7, 0.0, 0.3, pad=pad, in_place=True)
    M.close(got, *M.adjust_reference(scores, ids, None, None, allowed[:1], 0.7, 0.0, 0.3))


def test_clipping(ctx):
    sizes = [(3001, 2001, "f32", 3, 1), (90001, 37, "bf16", 1, 1), (5003, 1003, "bf16", 0, 0),
             (1, 100003, "f32", 0, 3)]
    a, g = _make(ctx, np.random.default_rng(6), sizes)
    norm = _norm(a)
    most = float(np.float32(norm / 3))
    outs = [M.blank(ctx, x.rows, x.cols, x.kind, x.pad, x.shift) for x in g]
    for entries, to in (([_entry(x, o) for x, o in zip(g, outs)], outs),
                        ([_entry(x, x) for x in g], g)):
        got = _clip(ctx, entries, most)
        assert abs(got - norm) <= norm * M.U * 1.001
        for x, m in zip(a, to):
            by = x * (most / norm)
            half = M.U + (D.HALF["bf16"] if m.kind == "bf16" else 0.0)
            full = D.decode(ctx.download(m.at, m.shift + m.rows * m.stride, M.DTYPE[m.kind]), m.kind)
            body = full[m.shift:].reshape(m.rows, m.stride)
            M.close(body[:, :m.cols], by, np.abs(by) * half * 1.001)
            between = body[:, m.cols:]
            assert np.all(np.isnan(between) if to is g else between == M.GUARD)

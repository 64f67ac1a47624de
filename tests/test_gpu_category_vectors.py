"""Category vectors and their gradient on the GPU, against plain 64-bit forms."""
import ctypes

import numpy as np
import pytest

import device_ops as D
import macboost_amd as mb
import model_ops as M

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = mb.Context(0)
    yield c
    c.close()


def _values(rng, rows, cols, kind):
    return D.rounded(rng.standard_normal((rows, cols)).astype(np.float32), kind)


def _ids(rng, rows, entries, skew=0.0, out=0.1):
    p = np.arange(1, entries + 1) ** -float(skew)
    ids = rng.permutation(entries)[rng.choice(entries, rows, p=p / p.sum())].astype(np.int32)
    bad = rng.random(rows) < out
    ids[bad] = rng.choice(np.array([-1, entries, -2 ** 31, 2 ** 31 - 1], np.int32), bad.sum())
    return ids


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,dim,entries,pad,shift", [
    (1, 1, 1, 0, 0), (1, 64, 5, 0, 0), (64, 37, 1003, 3, 0), (5, 64, 10, 8, 0), (1000, 100, 7, 4, 0),
    (257, 1024, 50, 0, 0), (3, 2001, 4, 7, 0), (300, 33, 20, 0, 1), (4099, 8, 100, 0, 8),
    (70, 19, 33, 5, 0)])
def test_lookup(ctx, kind, rows, dim, entries, pad, shift):
    rng = np.random.default_rng(rows + dim)
    ids = _ids(rng, rows, entries)
    table = _values(rng, entries, dim, kind)
    base = _values(rng, rows, dim, kind)
    scale = 0.37
    idev = ctx.upload(ids)
    used = np.unique(ids[(ids >= 0) & (ids < entries)])
    dirty = np.full_like(table, np.nan)                  # rows that no id names are not read
    dirty[used] = table[used]
    t = M.Matrix(ctx, dirty, kind, pad, shift, fill=np.nan)
    for b in (None, base):
        out = M.blank(ctx, rows, dim, kind, pad, shift)
        bm = None if b is None else M.Matrix(ctx, b, kind, pad, shift, fill=np.nan)
        ctx.call("mbk_embed", M.embed_shape(rows, entries, dim, kind, out.stride, t.stride, scale),
                 t.ptr, idev, None if b is None else bm.ptr, out.ptr)
        ctx.sync()
        M.close(out.read(), *M.embed_reference(table, ids, b, scale, kind))
    out = M.Matrix(ctx, base, kind, pad, shift)          # in place
    ctx.call("mbk_embed", M.embed_shape(rows, entries, dim, kind, out.stride, t.stride, scale),
             t.ptr, idev, out.ptr, out.ptr)
    ctx.sync()
    M.close(out.read(), *M.embed_reference(table, ids, base, scale, kind))


GRADS = [
    # rows, dim, entries, skew, pad, shift
    (1, 1, 1, 0, 0, 0), (1, 4, 300, 0, 0, 0), (2, 37, 3, 0, 3, 0), (63, 64, 5, 0, 0, 0),
    (64, 16, 1, 0, 0, 0), (65, 16, 1, 0, 0, 0), (200, 8, 2, 0, 0, 0), (129, 24, 129, 1, 0, 0),
    (1000, 100, 50, 1, 4, 0), (16384, 12, 700, 1, 0, 0), (16384, 5, 255, 0, 0, 0),
    (16385, 12, 700, 1, 0, 0), (20000, 37, 300, 0.5, 3, 0), (3000, 1030, 40, 1, 0, 0),
    (5000, 260, 9000, 1, 0, 1), (30000, 3, 100000, 1, 1, 0), (40000, 1, 2000000, 0, 0, 0),
    (600000, 2, 3000, 1.5, 0, 0), (2200000, 1, 70, 0, 0, 0), (50000, 70, 1, 0, 0, 0),
    (300, 2, 50000, 0, 0, 0), (17000, 2, 1100000, 0, 0, 0),
]


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,dim,entries,skew,pad,shift", GRADS)
def test_gradient(ctx, kind, rows, dim, entries, skew, pad, shift):
    rng = np.random.default_rng(rows * 3 + dim + entries)
    ids = _ids(rng, rows, entries, skew)
    dout = _values(rng, rows, dim, kind)
    base = _values(rng, entries, dim, kind)
    outside = (ids < 0) | (ids >= entries)
    scale = -1.7
    idev = ctx.upload(ids)
    dirty = np.where(outside[:, None], np.float32(np.nan), dout)    # reaches nothing
    g = M.Matrix(ctx, dirty, kind, pad, shift, fill=np.nan)
    b = M.Matrix(ctx, base, kind, pad, shift, fill=np.nan)
    for of, bp in ((None, None), (base, b.ptr)):
        want = M.embed_grad_reference(dout, ids, entries, of, scale, kind)
        first = None
        for _ in range(2):
            out = M.blank(ctx, entries, dim, kind, pad, shift)
            ctx.call("mbk_embed_grad",
                     M.embed_shape(rows, entries, dim, kind, g.stride, out.stride, scale), idev,
                     g.ptr, bp, out.ptr)
            ctx.sync()
            got = out.read()
            M.close(got, *want)
            assert first is None or np.array_equal(got, first)      # bit for bit
            first = got
    # on top of what is there; entries without rows are not read
    used = np.zeros(entries, bool)
    used[ids[~outside]] = True
    start = np.where(used[:, None], base, np.float32(np.nan))
    out = M.Matrix(ctx, start, kind, pad, shift)
    ctx.call("mbk_embed_grad", M.embed_shape(rows, entries, dim, kind, g.stride, out.stride, scale),
             idev, g.ptr, out.ptr, out.ptr)
    ctx.sync()
    value, tol = M.embed_grad_reference(dout, ids, entries, base, scale, kind)
    M.close(out.read(), np.where(used[:, None], value, np.nan), tol)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,dim,entries,skew,pad,shift", [
    (47, 8, 30, 0, 0, 0), (48, 8, 30, 0, 0, 0), (129, 37, 7, 1, 3, 1), (1000, 256, 1023, 0, 0, 0),
    (1000, 1000, 1, 0, 0, 0), (1000, 300, 1023, 1, 0, 0), (1000, 4, 1024, 0, 0, 0),
    (1025, 3, 1, 0, 0, 0), (1025, 37, 1023, 0, 1, 1), (1025, 37, 1024, 0, 0, 0),
    (1100, 257, 2, 0, 0, 0), (2000, 513, 9, 1, 3, 0), (1500, 1025, 1000, 0, 0, 0),
    (33000, 16, 31, 2, 0, 0), (33000, 15, 32, 1, 0, 1), (70000, 4, 33, 3, 0, 0),
    (70000, 1, 1023, 0, 0, 0), (262145, 8, 5, 0, 0, 0), (300000, 2, 400, 0.5, 1, 0),
])
def test_gradient_of_few_entries(ctx, kind, rows, dim, entries, skew, pad, shift):
    """Up to 1023 entries, in slices of 128 to 1024 rows."""
    test_gradient(ctx, kind, rows, dim, entries, skew, pad, shift)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,dim,entries,skew,pad,shift", [
    (1000, 37, 20000, 0, 3, 0), (1024, 5, 1024, 2, 0, 1), (1024, 300, 1500, 3, 0, 0),
    (1025, 8, 2000, 2, 0, 0), (4096, 6, 5000, 1, 1, 0), (4000, 64, 1025, 3, 0, 0),
    (4097, 70, 1024, 2, 0, 0), (6000, 1030, 40, 1, 0, 0), (9000, 2060, 200, 0, 0, 0),
])
def test_gradient_of_many_entries_or_columns(ctx, kind, rows, dim, entries, skew, pad, shift):
    """From 1024 entries, or 4 times 64 pieces of 16 bytes, on: one sorted list."""
    test_gradient(ctx, kind, rows, dim, entries, skew, pad, shift)


@pytest.mark.parametrize("rows", [0, 1, 100, 20000])
@pytest.mark.parametrize("entries", [1, 5000])
def test_gradient_without_rows_in_any_entry(ctx, rows, entries):
    ids = ctx.upload(np.full(max(1, rows), -1, np.int32))
    g = M.Matrix(ctx, np.full((max(1, rows), 9), np.nan, np.float32), "f32")
    rng = np.random.default_rng(1)
    base = rng.standard_normal((entries, 9)).astype(np.float32)
    b = M.Matrix(ctx, base, "f32")
    for bp, want in ((None, np.zeros_like(base)), (b.ptr, base)):
        out = M.blank(ctx, entries, 9, "f32")
        ctx.call("mbk_embed_grad", M.embed_shape(rows, entries, 9, "f32", 9, 9), ids, g.ptr, bp,
                 out.ptr)
        ctx.sync()
        assert np.array_equal(out.read(), want)
    ctx.call("mbk_embed_grad", M.embed_shape(rows, entries, 9, "f32", 9, 9), ids, g.ptr, b.ptr,
             b.ptr)
    ctx.sync()
    assert np.array_equal(b.read(), base)
    out = M.blank(ctx, max(1, rows), 9, "f32")
    ctx.call("mbk_embed", M.embed_shape(rows, entries, 9, "f32", 9, 9), b.ptr, ids, None, out.ptr)
    ctx.sync()
    assert np.all(out.read() == (0.0 if rows else M.GUARD))


@pytest.mark.parametrize("rows,entries", [(3000, 40), (40000, 900), (100000, 1500)])
def test_gradient_of_runs_around_the_workers_ends(ctx, rows, entries):
    """Entries of 60 to 70 rows, some of 1 and of hundreds, in the ids' order."""
    rng = np.random.default_rng(rows)
    sizes = rng.choice([1, 16, 60, 63, 64, 65, 66, 128, 129, 500], entries)
    ids = np.repeat(np.arange(entries), sizes)[:rows].astype(np.int32)
    rng.shuffle(ids)
    dout = rng.standard_normal((ids.size, 6)).astype(np.float32)
    g, idev = M.Matrix(ctx, dout, "f32"), ctx.upload(ids)
    want = M.embed_grad_reference(dout, ids, entries, None, 1.0, "f32")
    out = M.blank(ctx, entries, 6, "f32")
    ctx.call("mbk_embed_grad", M.embed_shape(ids.size, entries, 6, "f32", 6, 6), idev, g.ptr, None,
             out.ptr)
    ctx.sync()
    M.close(out.read(), *want)
    zero = M.Matrix(ctx, np.zeros((entries, 6), np.float32), "f32")
    ctx.call("mbk_embed_grad", M.embed_shape(ids.size, entries, 6, "f32", 6, 6), idev, g.ptr,
             zero.ptr, zero.ptr)
    ctx.sync()
    M.close(zero.read(), *want)


def test_gradient_against_differences(ctx):
    """<dout, lookup> changes by <dtable, change> as the table does: both are linear."""
    rng = np.random.default_rng(5)
    rows, dim, entries, scale = 500, 12, 30, 0.5
    ids = _ids(rng, rows, entries)
    dout = rng.integers(-8, 9, (rows, dim)).astype(np.float32)
    table = rng.integers(-8, 9, (entries, dim)).astype(np.float32)
    change = rng.integers(-2, 3, (entries, dim)).astype(np.float32)
    idev, g = ctx.upload(ids), M.Matrix(ctx, dout, "f32")
    sums = []
    for t in (table - change, table + change):
        tm, out = M.Matrix(ctx, t, "f32"), M.blank(ctx, rows, dim, "f32")
        ctx.call("mbk_embed", M.embed_shape(rows, entries, dim, "f32", dim, dim, scale), tm.ptr,
                 idev, None, out.ptr)
        ctx.sync()
        sums.append((dout.astype(np.float64) * out.read()).sum())
    out = M.blank(ctx, entries, dim, "f32")
    ctx.call("mbk_embed_grad", M.embed_shape(rows, entries, dim, "f32", dim, dim, scale), idev,
             g.ptr, None, out.ptr)
    ctx.sync()
    # small whole numbers: no rounding anywhere
    assert (sums[1] - sums[0]) / 2 == (out.read().astype(np.float64) * change).sum()

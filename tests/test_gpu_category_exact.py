"""Gradients of category vectors in whole numbers whose sums f32 holds without rounding, so that a
row that is lost, or taken twice, shows however long its entry is."""
import numpy as np
import pytest

import device_ops as D
import macboost_amd as mb
import model_ops as M
from test_gpu_category_vectors import _ids

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = mb.Context(0)
    yield c
    c.close()


def _whole(rng, rows, cols, most):
    return rng.integers(-most, most + 1, (rows, cols), dtype=np.int8).astype(np.float32)


def _check(ctx, kind, rows, dim, entries, skew, pad=0, most=4):
    """Without a base, with one, and on top of what is there."""
    rng = np.random.default_rng(rows + 7 * dim + entries)
    ids = _ids(rng, rows, entries, skew, 0.01)
    kept = (ids >= 0) & (ids < entries)
    count = np.bincount(ids[kept], minlength=entries)
    dout, base = _whole(rng, rows, dim, most), _whole(rng, entries, dim, 8)
    # halves of sums below 2^22, and a base of up to 8: 24 bits
    assert count.max() * most < 2 ** 22
    if dim > entries:
        total = np.stack([dout[ids == e].sum(0, dtype=np.float64) for e in range(entries)])
    else:
        total = np.stack([np.bincount(ids[kept], dout[kept, c], entries) for c in range(dim)], 1)
    dout[~kept] = np.nan
    idev, g = ctx.upload(ids), M.Matrix(ctx, dout, kind, pad, fill=np.nan)
    b = M.Matrix(ctx, base, kind, pad, fill=np.nan)
    shape = M.embed_shape(rows, entries, dim, kind, g.stride, dim + pad, -0.5)
    for of, bp in ((0.0, None), (base, b.ptr)):
        out = M.blank(ctx, entries, dim, kind, pad)
        ctx.call("mbk_embed_grad", shape, idev, g.ptr, bp, out.ptr)
        ctx.sync()
        assert np.array_equal(out.read(), D.rounded((total * -0.5 + of).astype(np.float32), kind))
    start = np.where(count[:, None] > 0, base, np.float32(np.nan))
    want = np.where(count[:, None] > 0, total * -0.5 + base, np.nan).astype(np.float32)
    out = M.Matrix(ctx, start, kind, pad)
    ctx.call("mbk_embed_grad", shape, idev, g.ptr, out.ptr, out.ptr)
    ctx.sync()
    assert np.array_equal(out.read(), D.rounded(want, kind), equal_nan=True)


@pytest.mark.parametrize("kind,rows,dim,entries,skew", [
    ("f32", 1048577, 4, 2000, 0), ("f32", 1048576, 1, 1024, 1), ("bf16", 1048580, 2, 70000, 0.5),
    ("bf16", 1100003, 8, 2000, 0), ("f32", 4300000, 13, 2000, 1),
])
def test_the_longest_lists_of_a_workgroup(ctx, kind, rows, dim, entries, skew):
    """From 2^20 rows of one to four pieces on, and their sort of several chunks a workgroup."""
    _check(ctx, kind, rows, dim, entries, skew)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,dim,entries,skew", [
    # slices, of one entry, of few and of many, narrow and wide
    (50000, 70, 1, 0), (262145, 8, 5, 0), (1000000, 1, 70, 0.5), (300000, 2, 400, 2),
    (70001, 36, 1023, 2), (2000, 513, 9, 1), (1100, 257, 2, 0), (6000, 250, 3, 0),
    # one launch, whose longest entries have workgroups of their own
    (1024, 300, 1500, 3), (1000, 20, 20000, 2), (1024, 1030, 1, 0),
    # a sort in one workgroup, and longer ones
    (4000, 64, 1025, 3), (4096, 2, 5000, 2), (20000, 300, 1100, 2), (100000, 37, 1500, 1.5),
    (200000, 16, 2000, 2), (600000, 2, 3000, 1.5), (600000, 5, 3000, 3),
    # rows of several wavefronts
    (9000, 2064, 30, 1), (6000, 1030, 40, 2), (9000, 2060, 200, 3),
])
def test_long_entries(ctx, kind, rows, dim, entries, skew):
    _check(ctx, kind, rows, dim, entries, skew, pad=rows % 3)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_sums_of_slices_beyond_their_limit(ctx, kind):
    """300 entries of 256 columns, whose slices' sums would take 90 MB: one sorted list."""
    _check(ctx, kind, 300000, 256, 300, 1)


@pytest.mark.parametrize("entries", [1, 1500])
def test_one_entry_of_2_to_21_rows(ctx, entries):
    """All rows but a few to one entry: more than 1,000 sums of slices or of workgroups."""
    _check(ctx, "f32", (1 << 21) + 1, 5, entries, 40, most=1)

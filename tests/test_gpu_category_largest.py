"""Category vectors, clipping, 4-bit scores and penalties at the ends of their sizes: 2^20 columns,
2^31 - 256 entries and classes, packed forms past 2^31 bytes."""
import ctypes

import numpy as np
import pytest

import device_ops as D
import macboost_amd as mb
import model_ops as M
from macboost_amd import _core
from test_gpu_category_exact import _check, _whole

pytestmark = pytest.mark.gpu

MOST = 2 ** 31 - 256


@pytest.fixture()
def ctx():
    c = mb.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,dim,entries", [(100, 1 << 20, 3), (70, (1 << 20) - 1, 2),
                                              (260, (1 << 20) - 3, 2), (1200, 100003, 4)])
def test_rows_of_2_to_20_columns(ctx, kind, rows, dim, entries):
    _check(ctx, kind, rows, dim, entries, 1.0)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,group,dim", [(1, 128, 1 << 20), (5, 32, (1 << 20) - 1), (40, 64, 1 << 20)])
def test_scores_of_2_to_20_columns(ctx, kind, rows, group, dim):
    """h of -1, 0 and 1, w whole numbers with a 7 in every group, so that its scale is 1: whole sums
    below 2^24."""
    rng = np.random.default_rng(rows)
    h, w = _whole(rng, rows, dim, 1), _whole(rng, 19, dim, 7)
    w[:, ::group] = 7
    want = h.astype(np.float64) @ w.astype(np.float64).T
    got = M.Fourbit(ctx, w, kind, group).scores(h, score_pad=1)
    assert np.array_equal(got, want.astype(np.float32))


@pytest.mark.parametrize("rows", [1000, 5000])
def test_2_to_31_entries(ctx, rows):
    """Every entry of the table is written, which the norm of all of them tells."""
    rng = np.random.default_rng(rows)
    ids = rng.integers(0, MOST, rows).astype(np.int32)
    ids[:8] = [0, MOST - 1, MOST - 1, 1 << 30, (1 << 30) + 1, -1, 2 ** 31 - 1, MOST - 2]
    dout = _whole(rng, rows, 1, 4)
    table = ctx.alloc(MOST * 2 + 128)
    idev, shape = ctx.upload(ids), M.embed_shape(rows, MOST, 1, "bf16", 1, 1)
    norm = ctx.upload(np.zeros(1, np.float32))
    all_of = ctx.tensors([(table, None, 1, MOST, MOST, _core.BF16)])
    kept = (ids >= 0) & (ids < MOST)
    for sign in (1, -1):
        g = M.Matrix(ctx, dout * sign, "bf16")
        ctx.call("mbk_embed_grad", shape, idev, g.ptr, None, table)
        ctx.call("mbk_grad_clip", all_of.ptr, np.inf, norm)
        used, at = np.unique(ids[kept], return_inverse=True)
        total = np.bincount(at, dout[kept, 0] * sign)
        ctx.sync()
        assert ctx.download(norm, 1, np.float32)[0] == np.float32(np.sqrt((total ** 2).sum()))
        out = M.blank(ctx, rows, 1, "bf16")              # and looked up
        ctx.call("mbk_embed", shape, table, idev, None, out.ptr)
        ctx.sync()
        want = np.zeros(rows)
        want[kept] = total[at]
        assert np.array_equal(out.read()[:, 0], want)
    # on top of what is there
    ctx.call("mbk_embed_grad", shape, idev, g.ptr, table, table)
    ctx.call("mbk_grad_clip", all_of.ptr, np.inf, norm)
    ctx.sync()
    assert ctx.download(norm, 1, np.float32)[0] == np.float32(2 * np.sqrt((total ** 2).sum()))
    all_of.close()


def _repeated(ctx, rows, table, kind):
    """[rows] of the table's rows, over and over, in device memory."""
    n, dim = table.shape
    t = M.Matrix(ctx, table, kind)
    ids = ctx.upload((np.arange(rows, dtype=np.int64) % n).astype(np.int32))
    out = ctx.alloc(rows * dim * M.SIZE[kind] + 128)
    ctx.call("mbk_embed", M.embed_shape(rows, n, dim, kind, dim, dim), t.ptr, ids, None, out)
    ctx.sync()
    return out


def test_2_to_31_classes_under_penalties(ctx):
    """In place, looked at around the history's classes and the ends of the mask's words."""
    period = np.random.default_rng(1).standard_normal((1, 1024)).astype(np.float32)
    scores = _repeated(ctx, 1 << 21, period, "f32")
    ids = np.array([[5, MOST - 1, 1 << 30, MOST - 1, 4095, 4096, 5, 5, 2 ** 31 - 1, -1]], np.int32)
    mask = np.full(MOST // 32, 0xFFFFFFFF, np.uint32)
    mask[[0, 1 << 20, MOST // 32 - 1]] = 0xF0F0FFFF
    shape = _core.MbkAdjustShape(1, MOST, MOST, MOST, ids.shape[1], ids.shape[1], 0, 1.5, 0.25, 0.5)
    ctx.call("mbk_adjust", ctypes.byref(shape), scores, ctx.upload(ids), None, None, ctx.upload(mask),
             scores)
    ctx.sync()
    for a in (0, 4064, (1 << 25) - 64, (1 << 30) - 64, MOST - 128):
        n = 128
        got = ctx.download(scores + a * 4, n, np.float32)
        was = np.resize(period[0], 1 << 12)[a % 1024:][:n][None]
        inside = ids[(ids >= a) & (ids < a + n)][None] - a
        M.close(got[None], *M.adjust_reference(was, inside, None, None,
                                               mask[None, a // 32:(a + n) // 32], 1.5, 0.25, 0.5))
    # behind the last class
    assert np.array_equal(ctx.download(scores + MOST * 4, 256, np.float32), period[0, MOST % 1024:])


def test_packed_class_vectors_past_2_to_31_bytes(ctx):
    classes, dim, n = (1 << 25) + 49, 32, 1009
    rng = np.random.default_rng(2)
    few = _whole(rng, n, dim, 7)
    few[:, 3] = 7                                        # scales of 1
    few[::5] *= 4                                        # and of 4
    w = _repeated(ctx, classes, few, "bf16")
    shape = _core.MbkFourbitShape(classes, dim, 32)
    size = _core.fourbit_bytes(shape)
    assert size > 2 ** 31
    packed = ctx.alloc(size)
    ctx.call("mbk_fourbit_pack", ctypes.byref(shape), _core.BF16, w, dim, packed)
    for rows in (2, 35):                                 # held in LDS, and tiles of classes
        h = _whole(rng, rows, dim, 8)
        hm = M.Matrix(ctx, h, "bf16")
        scores = ctx.alloc(rows * classes * 4 + 256)
        ctx.call("mbk_fourbit_scores", ctypes.byref(shape), rows, _core.BF16, hm.ptr, dim, packed, None,
                 scores, classes)
        ctx.sync()
        want = (h.astype(np.float64) @ few.T.astype(np.float64)).astype(np.float32)
        for r in (0, 1, rows - 1):
            got = ctx.download(scores + r * classes * 4, classes, np.float32)
            whole = classes // n * n
            assert np.all(got[:whole].reshape(-1, n) == want[r])
            assert np.array_equal(got[whole:], want[r, :classes - whole])

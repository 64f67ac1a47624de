"""The operators over arrays past 2^31 elements and launches past 2^32 threads.  Only rows
at the two ends are written and compared; what lies between is whatever the memory held."""
import ctypes

import numpy as np
import pytest

import device_ops as D
import macboost_amd as mb
from macboost_amd import _core

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture
def ctx():
    c = mb.Context(0)
    yield c
    c.close()


def _put(ctx, at, a):
    a = np.ascontiguousarray(a)
    err = ctypes.c_char_p()
    ctx._check(_core.lib().mbk_copy_to_device(ctx.ptr, at, a.ctypes.data, a.nbytes,
                                              ctypes.byref(err)), err)


@pytest.mark.parametrize("major,blocked", [("row", False), ("feature", True), ("row", True),
                                           ("feature", False)])
def test_rows_by_expert_past_2_to_31_elements(ctx, major, blocked):
    rows, cols, ends = 2_200_000, 1000, 20
    rng = np.random.default_rng(5)
    expert = rng.integers(0, 3, (rows, 1)).astype(np.int32)
    s = D.Experts(ctx, expert, 3)
    s.sort()
    offsets, _, slot = D.sort_reference(expert, 3)
    spot = np.r_[0:ends, rows - ends:rows]
    values = rng.standard_normal((2 * ends, cols)).astype(np.float32)
    total = rows * cols * 4
    x, sorted_x, back, d_sorted = (ctx.alloc(total) for _ in range(4))
    d_weights = ctx.alloc(rows * 4)
    stride = (cols, 1) if major == "row" else (1, rows)

    def matrix(p):
        return ctypes.byref(_core.MbkExpertMatrix(p, *stride, cols, _core.F32, int(blocked)))

    def read_row(p, i):
        if major == "row":
            return ctx.download(p + i * cols * 4, cols, np.float32)
        return np.concatenate([ctx.download(p + (f * rows + i) * 4, 1, np.float32)
                               for f in range(0, cols, 37)])

    def read_slot(p, s):
        if not blocked:
            return ctx.download(p + s * cols * 4, cols, np.float32)
        e = int(np.searchsorted(offsets, s, "right")) - 1
        first, n = int(offsets[e]), int(offsets[e + 1] - offsets[e])
        return np.concatenate([ctx.download(p + (cols * first + f * n + s - first) * 4, 1,
                                            np.float32) for f in range(0, cols, 37)])

    every = slice(None, None, 37)
    for n, i in enumerate(spot):
        if major == "row":
            _put(ctx, x + int(i) * cols * 4, values[n])
    if major == "feature":
        for f in range(cols):
            _put(ctx, x + f * rows * 4, values[:ends, f])
            _put(ctx, x + (f * rows + rows - ends) * 4, values[ends:, f])
    ctx.call("mbk_expert_gather", ctypes.byref(s.plan), matrix(x), sorted_x)
    ctx.call("mbk_expert_combine", ctypes.byref(s.plan), sorted_x, None, matrix(back))
    ctx.call("mbk_expert_combine_grad", ctypes.byref(s.plan), matrix(x), sorted_x, None, d_sorted,
             d_weights)
    ctx.sync()
    for n, i in enumerate(spot):
        at = int(slot[i, 0])
        want = values[n] if not blocked else values[n][every]
        assert np.array_equal(read_slot(sorted_x, at), want)
        assert np.array_equal(read_slot(d_sorted, at), want)
        assert np.array_equal(read_row(back, int(i)),
                              values[n] if major == "row" else values[n][every])
        exact = float((values[n].astype(np.float64) ** 2).sum())
        got = float(ctx.download(d_weights + int(i) * 4, 1, np.float32)[0])
        assert abs(got - exact) <= exact * cols * U


def test_rows_by_expert_past_2_to_32_threads(ctx):
    rows, ends = (1 << 30) + (1 << 26), 1000            # 64 rows a workgroup of 256
    expert = ctx.upload(np.zeros(rows, np.int32))
    offsets, source, slot = ctx.alloc(8), ctx.alloc(rows * 4), ctx.alloc(rows * 4)
    plan = _core.MbkExpertPlan(rows, 1, 1, expert, offsets, source, slot)
    x, sorted_x, back = (ctx.alloc(rows * 4) for _ in range(3))
    first, last = np.arange(ends, dtype=np.float32), -np.arange(ends, dtype=np.float32)
    _put(ctx, x, first)
    _put(ctx, x + (rows - ends) * 4, last)
    m = lambda p: ctypes.byref(_core.MbkExpertMatrix(p, 1, rows, 1, _core.F32, 0))
    ctx.call("mbk_expert_sort", ctypes.byref(plan))
    ctx.call("mbk_expert_gather", ctypes.byref(plan), m(x), sorted_x)
    ctx.call("mbk_expert_combine", ctypes.byref(plan), sorted_x, None, m(back))
    ctx.sync()
    assert list(ctx.download(offsets, 2, np.int32)) == [0, rows]
    tail = np.arange(rows - ends, rows)
    for a in (source, slot):
        assert np.array_equal(ctx.download(a + (rows - ends) * 4, ends, np.int32), tail)
    for a in (sorted_x, back):
        assert np.array_equal(ctx.download(a, ends, np.float32), first)
        assert np.array_equal(ctx.download(a + (rows - ends) * 4, ends, np.float32), last)


# 67M rows: a wavefront a row joins their sums
@pytest.mark.parametrize("rows,d", [(17_000_000, 128), ((1 << 26) + 1000, 130)])
def test_xent_past_2_to_31_elements(ctx, rows, d):
    classes, ends = 3, 100
    rng = np.random.default_rng(d)
    w = rng.standard_normal((classes, d)).astype(np.float32)
    bias = rng.standard_normal(classes).astype(np.float32)
    labels = rng.integers(0, classes, rows, dtype=np.int32)
    h = rng.standard_normal((2 * ends, d)).astype(np.float32)
    spot = np.r_[0:ends, rows - ends:rows]
    r = D.xent_reference(h, w, labels[spot], "bf16", bias)
    hdev, dh = ctx.alloc(rows * d * 2), ctx.alloc(rows * d * 2)
    _put(ctx, hdev, D.encode(h[:ends], "bf16"))
    _put(ctx, hdev + (rows - ends) * d * 2, D.encode(h[ends:], "bf16"))
    loss, lse = ctx.alloc(rows * 4), ctx.alloc(rows * 4)
    shape = _core.MbkXentShape(rows, classes, d, _core.BF16, d, d)
    ctx.call("mbk_xent_grad", ctypes.byref(shape), hdev, ctx.upload(D.encode(w, "bf16")),
             ctx.upload(bias), ctx.upload(labels), None, loss, lse, dh, None, None)
    ctx.sync()

    def both(p, shape, dtype, size):
        return np.concatenate([ctx.download(p, shape, dtype),
                               ctx.download(p + (rows - ends) * size, shape, dtype)])

    D.check({"loss": both(loss, ends, np.float32, 4), "lse": both(lse, ends, np.float32, 4),
             "dh": D.decode(both(dh, (ends, d), np.uint16, d * 2), "bf16")}, r,
            ("loss", "lse", "dh"))

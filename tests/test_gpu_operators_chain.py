"""A boosting round of several outputs without experts: forests' outputs, a column at a time, to
the row-major h of the many-class loss, and its dh back to columns that are quantised."""
import ctypes

import numpy as np
import pytest

import device_ops as D
from macboost_amd import _core
from test_gpu_operators import _leaf_forest, _predict_reference, ctx      # noqa: F401

pytestmark = pytest.mark.gpu


def test_a_round_of_one_booster_of_several_outputs(ctx):
    rows, cols, dim, classes, trees = 700, 5, 3, 60, 4
    rng = np.random.default_rng(78)
    x = rng.random((rows, cols)).astype(np.float32)
    w = rng.standard_normal((classes, dim)).astype(np.float32)
    y = rng.integers(0, classes, rows).astype(np.int32)
    forests = [_leaf_forest(rng, trees, cols) for _ in range(dim)]
    xdev = ctx.upload(np.ascontiguousarray(x.T))
    outputs = ctx.alloc(dim * rows * 4)
    for j in range(dim):
        f = {key: ctx.upload(v) for key, v in forests[j].items()}
        ctx.call("mbk_predict_forest", f["feature"], f["threshold"], f["flags"], f["leaf"], None,
                 trees, 3, xdev, rows, 255, 0.0, outputs + j * rows * 4)
    s = D.Experts(ctx, np.zeros((rows, 1), np.int32), 1)
    s.sort()
    loss = D.Xent(ctx, np.zeros((rows, dim), np.float32), w, y, "f32")
    hm = _core.MbkExpertMatrix(loss.h, dim, 1, dim, _core.F32, 1)
    dm = _core.MbkExpertMatrix(loss.dh, dim, 1, dim, _core.F32, 1)
    columns = ctx.alloc(dim * rows * 4)
    ctx.call("mbk_expert_combine", ctypes.byref(s.plan), outputs, None, ctypes.byref(hm))
    loss.grad()
    ctx.call("mbk_expert_gather", ctypes.byref(s.plan), ctypes.byref(dm), columns)
    got = loss.results()
    h = ctx.download(loss.h, (rows, dim), np.float32)
    assert np.array_equal(h.T, ctx.download(outputs, (dim, rows), np.float32))
    per = np.stack([_predict_reference(f, x) for f in forests], 1)
    assert np.all(np.abs(h - per) <= np.abs(per) * 2.0 ** -24)
    D.check(got, D.xent_reference(h, w, y, "f32"))
    assert np.array_equal(ctx.download(columns, (dim, rows), np.float32), got["dh"].T)
    zeros, entries, maxima = ctx.upload(np.zeros(rows, np.float32)), ctx.alloc(rows * 8), ctx.alloc(8)
    for j in range(dim):
        ctx.call("mbk_quantize", 0, 0.0, 0.0, columns + j * rows * 4, zeros, None, rows, maxima,
                 entries)
        ctx.sync()
        assert ctx.download(maxima, 2, np.float32)[0] == np.abs(got["dh"][:, j]).max()

"""A boosting round of several outputs with category vectors: forests' outputs to h, each row's
category vector on top of it in place, the many-class loss, the vectors' gradient and the clipping, and
dh back to columns that are quantised for the next trees; then the answers of the trained model."""
import ctypes

import numpy as np
import pytest

import device_ops as D
import model_ops as M
from macboost_amd import _core
from test_gpu_operators import _leaf_forest, _predict_reference, ctx      # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,dim,classes,entries", [(700, 3, 60, 40), (20011, 5, 300, 2000)])
def test_a_round_of_forests_and_category_vectors(ctx, rows, dim, classes, entries):
    cols, trees, ref = 5, 4, ctypes.byref
    rng = np.random.default_rng(rows)
    x = rng.random((rows, cols)).astype(np.float32)
    w = rng.standard_normal((classes, dim)).astype(np.float32)
    table = rng.standard_normal((entries, dim)).astype(np.float32)
    y = rng.integers(0, classes, rows).astype(np.int32)
    ids = rng.integers(-1, entries, rows).astype(np.int32)
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
    columns, tdev, idev = ctx.alloc(dim * rows * 4), ctx.upload(table), ctx.upload(ids)
    dtable, norm = M.blank(ctx, entries, dim, "f32"), ctx.upload(np.zeros(1, np.float32))
    grads = ctx.tensors([(loss.dw, loss.dw, classes, dim, dim, _core.F32),
                         (loss.db, loss.db, 1, classes, classes, _core.F32),
                         (dtable.ptr, dtable.ptr, entries, dim, dim, _core.F32)])
    ctx.call("mbk_expert_combine", ref(s.plan), outputs, None, ref(hm))
    vectors = M.embed_shape(rows, entries, dim, "f32", dim, dim, 0.5)
    ctx.call("mbk_embed", vectors, tdev, idev, loss.h, loss.h)
    loss.grad()
    ctx.call("mbk_embed_grad", vectors, idev, loss.dh, None, dtable.ptr)
    got = loss.results()
    got["dtable"] = dtable.read().copy()
    ctx.call("mbk_grad_clip", grads.ptr, 0.25, norm)
    ctx.call("mbk_expert_gather", ref(s.plan), ref(dm), columns)
    ctx.sync()

    h = ctx.download(loss.h, (rows, dim), np.float32)
    per = ctx.download(outputs, (dim, rows), np.float32).T
    exact = np.stack([_predict_reference(f, x) for f in forests], 1)
    assert np.all(np.abs(per - exact) <= np.abs(exact) * M.U)
    M.close(h, *M.embed_reference(table, ids, per, 0.5, "f32"))
    D.check(got, D.xent_reference(h, w, y, "f32"))
    M.close(got["dtable"], *M.embed_grad_reference(got["dh"], ids, entries, None, 0.5, "f32"))
    parts = [got["dw"], got["db"][None], got["dtable"]]
    size = np.sqrt(sum((g.astype(np.float64) ** 2).sum() for g in parts))
    assert abs(ctx.download(norm, 1, np.float32)[0] - size) <= size * M.U * 1.001
    clipped = loss.results()
    for g, after in zip(parts, (clipped["dw"], clipped["db"][None], dtable.read())):
        by = g * min(1.0, 0.25 / size)
        M.close(after, by, np.abs(by) * M.U * 1.001 + 1e-44)
    # dh is not on the list: its columns are the next trees' gradients
    assert np.array_equal(ctx.download(columns, (dim, rows), np.float32), got["dh"].T)
    zeros, rows_of, maxima = ctx.upload(np.zeros(rows, np.float32)), ctx.alloc(rows * 8), ctx.alloc(8)
    for j in range(dim):
        ctx.call("mbk_quantize", 0, 0.0, 0.0, columns + j * rows * 4, zeros, None, rows, maxima,
                 rows_of)
        ctx.sync()
        assert ctx.download(maxima, 2, np.float32)[0] == np.abs(got["dh"][:, j]).max()

    # answers: scores with W in 4 bits, under what each row has had
    shape = _core.MbkFourbitShape(classes, dim, 32)
    packed, scores = ctx.alloc(_core.fourbit_bytes(shape)), M.blank(ctx, rows, classes, "f32")
    ctx.call("mbk_fourbit_pack", ref(shape), _core.F32, loss.w, dim, packed)
    ctx.call("mbk_fourbit_scores", ref(shape), rows, _core.F32, loss.h, dim, packed, None, scores.ptr,
             classes)
    ctx.sync()
    z = scores.read().copy()
    M.close(z, *M.scores_reference(h, M.values(*M.quantised(w, 32), dim), None, "f32"))
    rule = _core.MbkAdjustShape(rows, classes, classes, classes, 1, 1, 0, 1.0, 1.5, 0.0)
    ctx.call("mbk_adjust", ref(rule), scores.ptr, loss.labels, None, None, None, scores.ptr)
    ctx.sync()
    M.close(scores.read(), *M.adjust_reference(z, y[:, None], None, None, None, 1.0, 1.5, 0.0))
    grads.close()

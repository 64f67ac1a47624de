"""Scores from class vectors in 4 bits on the GPU, against plain 64-bit forms."""
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


def _problem(seed, rows, dim, classes, kind):
    rng = np.random.default_rng(seed)
    h = D.rounded(rng.standard_normal((rows, dim)).astype(np.float32), kind)
    w = D.rounded((rng.standard_normal((classes, dim)) / np.sqrt(dim)).astype(np.float32), kind)
    return rng, h, w


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("classes,dim,pad", [(1, 1, 0), (16, 128, 0), (17, 129, 3), (100, 300, 0),
                                             (33, 31, 1), (5, 1000, 0)])
def test_pack(ctx, kind, group, classes, dim, pad):
    _, _, w = _problem(classes + dim, 1, dim, classes, kind)
    w[classes // 2] *= 1e-30                              # a class of another size
    w = D.rounded(w, kind)
    w[0, :min(dim, 64)] = 0
    code, scale = M.quantised(w, group)
    got_code, got_scale = M.Fourbit(ctx, w, kind, group, pad).read()
    width = code.shape[1]
    assert np.array_equal(got_code[:classes, :width], code)
    assert not got_code[classes:].any() and not got_code[:classes, width:].any()
    assert np.array_equal(got_scale[:classes, :scale.shape[1]], scale.astype(np.float64))
    assert not got_scale[classes:].any() and not got_scale[:classes, scale.shape[1]:].any()


def test_pack_ties_and_ends_of_the_codes(ctx):
    w = np.zeros((3, 32), np.float32)
    w[0, :] = (np.arange(32) - 16) / 2                    # the scale is 8/7 in bf16
    w[1, :16] = np.linspace(-7, 7, 16)
    w[1, 20] = 7
    w[2, :8] = [7, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5, -7]   # a scale of 1: ties to even
    code, scale = M.quantised(w, 32)
    assert scale[2, 0] == 1 and list(code[2, :8]) == [7, 0, 2, 2, 0, -2, -2, -7]
    got, _ = M.Fourbit(ctx, w, "f32", 32).read()
    assert np.array_equal(got[:3, :32], code)


SHAPES = [
    # rows, dim, classes
    (1, 1, 1), (1, 64, 1000), (2, 37, 100), (3, 128, 16), (8, 200, 31), (9, 129, 333), (15, 96, 47),
    (16, 1024, 500), (17, 1000, 129), (31, 300, 65), (33, 260, 1003), (64, 512, 200), (65, 130, 77),
    (130, 777, 300), (201, 100, 2100), (500, 33, 40), (4, 4000, 50), (1, 8200, 18),
    (40, 1300, 70), (16, 2600, 300), (20, 2600, 33), (96, 140, 600), (5, 1024, 2000), (7, 600, 5000),
]


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,dim,classes", SHAPES)
def test_scores(ctx, kind, rows, dim, classes):
    rng, h, w = _problem(rows + dim + classes, rows, dim, classes, kind)
    bias = rng.standard_normal(classes).astype(np.float32)
    bias[rng.random(classes) < 0.1] = -np.inf
    group = (32, 64, 128)[(rows + dim) % 3]
    q = M.Fourbit(ctx, w, kind, group)
    held = M.values(*M.quantised(w, group), dim)
    M.close(q.scores(h), *M.scores_reference(h, held, None, kind))
    got = q.scores(h, bias, pad=3, score_pad=5)
    M.close(got, *M.scores_reference(h, held, bias, kind))
    assert np.array_equal(got, q.scores(h, bias, pad=8, score_pad=4))       # bit for bit


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows,dim,classes", [(1, 1024, 20000), (16, 256, 9000), (40, 520, 5000),
                                              (300, 384, 4000)])
def test_scores_of_many_classes(ctx, kind, group, rows, dim, classes):
    rng, h, w = _problem(rows + group, rows, dim, classes, kind)
    q = M.Fourbit(ctx, w, kind, group)
    held = M.values(*M.quantised(w, group), dim)
    M.close(q.scores(h), *M.scores_reference(h, held, None, kind))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_scores_of_rows_in_turns(ctx, kind):
    """More columns of h than are held at a time."""
    rows, dim, classes = 16384 + 50, 4, 20
    rng, h, w = _problem(3, rows, dim, classes, kind)
    held = M.values(*M.quantised(w, 32), dim)
    M.close(M.Fourbit(ctx, w, kind, 32).scores(h), *M.scores_reference(h, held, None, kind))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("size", [1e-38, 1e-20, 1e20, 1e37])
def test_scores_of_any_magnitude(ctx, kind, size):
    rng, h, w = _problem(7, 20, 200, 60, kind)
    h[3] = D.rounded(h[3] * np.float32(size), kind)
    h[4] = 0
    w[5] = D.rounded(w[5] * np.float32(size), kind)
    w[6] = 0
    held = M.values(*M.quantised(w, 64), 200)
    with np.errstate(over="ignore"):
        want, tol = M.scores_reference(h, held, None, kind)
        want = np.where(np.abs(want) > 3.4028235e38, np.sign(want) * np.inf, want)
    # results below f32's normal range have a step of 2^-149
    M.close(M.Fourbit(ctx, w, kind, 64).scores(h), want, tol + 2.0 ** -149)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_rows_and_classes_that_are_not_finite_stay_apart(ctx, kind):
    rng, h, w = _problem(8, 20, 100, 40, kind)
    h[3, 50], h[4, 0], h[5, 99] = np.inf, np.nan, -np.inf
    w[7, 3], w[8, 99] = np.nan, np.inf
    bias = np.zeros(40, np.float32)
    bias[[8, 20]] = -np.inf
    got = M.Fourbit(ctx, w, kind, 32).scores(h, bias)
    rows, classes = np.ones(20, bool), np.ones(40, bool)
    rows[3:6], classes[7:9] = False, False
    held = M.values(*M.quantised(w[classes], 32), 100)
    want, tol = M.scores_reference(h[rows], held, bias[classes], kind)
    M.close(got[rows][:, classes], want, tol)
    assert np.all(got[:, [8, 20]] == -np.inf)            # not offered, whatever else
    open_ = np.isfinite(bias)
    assert not np.isfinite(got[3:6][:, open_]).any()
    assert np.isnan(got[:, 7]).all()


def test_elements_of_very_different_sizes(ctx):
    """Beside a row's or a class's largest element the others keep their bits."""
    rng, h, w = _problem(9, 4, 256, 32, "f32")
    h[:, 0] *= 2.0 ** 20
    w[:, :32] *= 2.0 ** -15
    w[:, 0] = 0                                          # the large one meets no weight
    held = M.values(*M.quantised(w, 32), 256)
    z, _ = M.scores_reference(h, held, None, "f32")
    size = np.abs(h[:, 1:]).astype(np.float64) @ np.abs(held[:, 1:]).T
    tol = size * ((2 * 383 + 16) * M.U + 2.0 ** -22) + \
        np.abs(h).max(1)[:, None] * 2.0 ** -49 * np.abs(held).sum(1)[None] + np.abs(z) * M.U
    M.close(M.Fourbit(ctx, w, "f32", 32).scores(h), z, tol)


def test_no_rows(ctx):
    _, h, w = _problem(1, 1, 10, 20, "f32")
    q = M.Fourbit(ctx, w, "f32", 32)
    out = M.blank(ctx, 1, 20, "f32")
    import ctypes
    ctx.call("mbk_fourbit_scores", ctypes.byref(q.shape), 0, 0, None, 10, q.packed, None, None, 20)
    ctx.sync()
    assert np.all(out.read() == M.GUARD)

"""The seam's operators on the GPU, against plain 64-bit forms: the loss over many
classes with its gradient, rows sorted by expert and back, and a boosting round that
uses them together.  Tolerances are half steps of rounding carried through the
formulas (device_ops.xent_reference)."""
import ctypes

import numpy as np
import pytest

import device_ops as D
import macboost_amd as mb
from macboost_amd import _core

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = mb.Context(0)
    yield c
    c.close()


def _problem(seed, n, d, v, scale=2.0):
    rng = np.random.default_rng(seed)
    h = rng.standard_normal((n, d)).astype(np.float32)
    w = (rng.standard_normal((v, d)) * scale / np.sqrt(d)).astype(np.float32)
    return rng, h, w, rng.integers(0, v, n).astype(np.int32)


# ---- the loss over many classes ----------------------------------------------------

SIZES = [(1, 1, 1), (1, 64, 1000), (2, 5, 3), (17, 33, 129), (128, 64, 128), (129, 65, 257),
         (300, 37, 1003), (257, 128, 640), (5, 257, 2000), (700, 100, 500), (64, 300, 4097),
         (1000, 16, 20), (40, 1024, 300)]


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("n,d,v", SIZES)
def test_xent_sizes(ctx, kind, n, d, v):
    rng, h, w, y = _problem(n * 7919 + d * 31 + v, n, d, v)
    bias = rng.standard_normal(v).astype(np.float32)
    weights = (rng.random(n) + 0.5).astype(np.float32)
    x = D.Xent(ctx, h, w, y, kind, bias, weights, h_pad=3, w_pad=5)
    want = D.xent_reference(h, w, y, kind, bias, weights)
    x.forward()
    D.check(x.results(False), want, ("loss", "lse"))
    x.grad()
    D.check(x.results(), want)


@pytest.mark.parametrize("kind,n,d,v", [
    ("f32", 2100, 200, 8200), ("bf16", 2100, 200, 8200),        # tiles that fill the chip
    ("f32", 33000, 130, 200), ("bf16", 33000, 130, 200),        # rows in two pieces
    ("f32", 5, 129, 1048576 + 700),                             # classes in two pieces
    ("f32", 9000, 20, 700), ("bf16", 70, 100, 30000)])
def test_xent_many_rows_or_classes(ctx, kind, n, d, v):
    rng, h, w, y = _problem(n + v, n, d, v)
    bias = rng.standard_normal(v).astype(np.float32)
    weights = (rng.random(n) + 0.5).astype(np.float32)
    y[::17] = -1
    x = D.Xent(ctx, h, w, y, kind, bias, weights)
    x.grad()
    D.check(x.results(), D.xent_reference(h, w, y, kind, bias, weights))


@pytest.mark.parametrize("kind,d", [("f32", 1), ("f32", 4), ("f32", 64), ("f32", 99), ("f32", 512),
                                    ("bf16", 1), ("bf16", 8), ("bf16", 66), ("bf16", 199),
                                    ("bf16", 200), ("bf16", 1024)])
@pytest.mark.parametrize("n,v", [(1, 1), (1, 1000), (3, 33), (16, 5000), (32, 30000), (32, 300)])
def test_xent_loss_of_few_rows(ctx, kind, d, n, v):
    rng, h, w, y = _problem(n + v + d, n, d, v)
    bias = rng.standard_normal(v).astype(np.float32)
    weights = (rng.random(n) + 0.5).astype(np.float32)
    closed = rng.random(v) < 0.2
    closed[0] = False
    open_classes = np.flatnonzero(~closed)
    y = open_classes[rng.integers(0, open_classes.size, n)].astype(np.int32)
    bias[closed] = -np.inf
    y[n // 2] = -1
    weights[n // 3] = 0
    want = D.xent_reference(h, w, y, kind, bias, weights)
    w[closed] = np.nan                   # not read
    h[n // 2] = np.inf
    x = D.Xent(ctx, h, w, y, kind, bias, weights, h_pad=3, w_pad=8)
    x.forward()
    got = x.results(False)
    keep = np.arange(n) != n // 2
    got["lse"], want["lse"] = got["lse"][keep], tuple(t[keep] for t in want["lse"])
    D.check(got, want, ("loss", "lse"))
    # without bias and weights
    _, h, w, y = _problem(n + v + d, n, d, v)
    x = D.Xent(ctx, h, w, y, kind)
    x.forward()
    D.check(x.results(False), D.xent_reference(h, w, y, kind), ("loss", "lse"))


# tiles of 256 x 256 in the scores, and in dh or in dW
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("n,v", [(16300, 1000), (1000, 16300)])
def test_xent_wide_tiles(ctx, kind, n, v):
    rng, h, w, y = _problem(n + 5 * v, n, 1000, v)
    bias = rng.standard_normal(v).astype(np.float32)
    bias[1::5] = -np.inf
    y[::17] = -1
    x = D.Xent(ctx, h, w, y, kind, bias)
    x.grad()
    D.check(x.results(), D.xent_reference(h, w, y, kind, bias))


@pytest.mark.parametrize("kind,d", [("f32", 1), ("f32", 31), ("f32", 96), ("f32", 130), ("f32", 512),
                                    ("bf16", 1), ("bf16", 40), ("bf16", 66), ("bf16", 199),
                                    ("bf16", 1024)])
@pytest.mark.parametrize("n,v", [(1, 1), (1, 1000), (7, 33), (32, 9000), (31, 300)])
def test_xent_gradient_of_few_rows(ctx, kind, d, n, v):
    rng, h, w, y = _problem(n + 3 * v + d, n, d, v)
    bias = rng.standard_normal(v).astype(np.float32)
    weights = (rng.random(n) + 0.5).astype(np.float32)
    closed = rng.random(v) < 0.2
    closed[0] = False
    open_classes = np.flatnonzero(~closed)
    y = open_classes[rng.integers(0, open_classes.size, n)].astype(np.int32)
    bias[closed] = -np.inf
    out = n // 2
    if n > 1:
        y[out] = -1
        weights[n // 3] = 0
    want = D.xent_reference(h, w, y, kind, bias, weights)
    w[closed] = np.nan                   # not read
    if n > 1:
        h[out] = np.inf
    x = D.Xent(ctx, h, w, y, kind, bias, weights, h_pad=3, w_pad=8)
    x.grad()
    got = x.results()
    first = {key: np.array(value) for key, value in got.items()}
    if n > 1:
        keep = np.arange(n) != out
        got["lse"], want["lse"] = got["lse"][keep], tuple(t[keep] for t in want["lse"])
        assert not got["dh"][out].any() and not got["dh"][n // 3].any()
    D.check(got, want)
    assert not got["dw"][closed].any() and not got["db"][closed].any()
    x.grad()
    for key, value in x.results().items():
        assert np.array_equal(np.array(value), first[key], equal_nan=True)
    # one gradient alone, without bias and weights
    _, h, w, y = _problem(n + 3 * v + d, n, d, v)
    want = D.xent_reference(h, w, y, kind)
    for alone in ("dh", "dw", "db"):
        x = D.Xent(ctx, h, w, y, kind)
        x.grad(**{key: key == alone for key in ("dh", "dw", "db")})
        D.check(x.results(), want, ("loss", "lse", alone))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("h_pad,w_pad", [(0, 0), (8, 0), (0, 8), (1, 2)])
def test_xent_strides_and_no_bias(ctx, kind, h_pad, w_pad):
    _, h, w, y = _problem(5, 200, 96, 384)
    x = D.Xent(ctx, h, w, y, kind, h_pad=h_pad, w_pad=w_pad)
    x.grad()
    D.check(x.results(), D.xent_reference(h, w, y, kind))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("d", [40, 300])
def test_xent_rows_out_and_classes_not_offered_reach_nothing(ctx, kind, d):
    rng, h, w, y = _problem(11, 150, d, 333)
    bias = rng.standard_normal(333).astype(np.float32)
    closed = rng.random(333) < 0.3
    closed[5] = False
    open_classes = np.flatnonzero(~closed)
    y = open_classes[rng.integers(0, open_classes.size, 150)].astype(np.int32)
    bias[closed] = -np.inf
    weights = (rng.random(150) + 0.5).astype(np.float32)
    y[[3, 149]] = -1
    y[4] = 333
    y[5] = np.iinfo(np.int32).max
    y[6] = np.iinfo(np.int32).min
    weights[7] = 0.0
    out = [3, 4, 5, 6, 7, 149]
    want = D.xent_reference(h, w, y, kind, bias, weights)
    # what must not be read: NaN, infinity and huge values
    h2, w2 = h.copy(), w.copy()
    h2[3], h2[4], h2[5], h2[7] = np.nan, np.inf, 3e38, -np.inf
    w2[closed] = np.resize(np.array([np.nan, np.inf, -np.inf, 1e38], np.float32),
                           (int(closed.sum()), 1))
    x = D.Xent(ctx, h2, w2, y, kind, bias, weights)
    x.grad()
    got = x.results()
    keep = np.ones(150, bool)
    keep[[3, 4, 5, 7]] = False
    got["lse"], want["lse"] = got["lse"][keep], tuple(t[keep] for t in want["lse"])
    D.check(got, want)
    assert np.all(got["loss"][out] == 0) and np.all(got["dh"][out] == 0)
    assert np.all(got["dw"][closed] == 0) and np.all(got["db"][closed] == 0)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("d", [24, 200])
def test_xent_no_class_offered(ctx, kind, d):
    _, h, w, y = _problem(12, 30, d, 70)
    h[3] = np.nan
    x = D.Xent(ctx, h, w, y, kind, np.full(70, -np.inf, np.float32))
    x.grad()
    r = x.results()
    assert np.all(r["lse"][np.arange(30) != 3] == -np.inf)
    for name in ("loss", "dh", "dw", "db"):
        assert np.all(r[name] == 0), name


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("d", [24, 200])
def test_xent_label_not_offered(ctx, kind, d):
    """Its loss is infinite; the gradient still pushes the other classes down."""
    rng, h, w, y = _problem(13, 20, d, 50)
    bias = np.zeros(50, np.float32)
    bias[7] = -np.inf
    y[y == 7] = 8
    want = D.xent_reference(h, w, y, kind, bias)
    y2 = y.copy()
    y2[4] = 7
    x = D.Xent(ctx, h, w, y2, kind, bias)
    x.grad()
    r = x.results()
    assert r["loss"][4] == np.inf
    keep = np.arange(20) != 4
    for name in ("loss", "lse", "dh"):
        r[name], want[name] = r[name][keep], tuple(t[keep] for t in want[name])
    D.check(r, want, ("loss", "lse", "dh"))
    assert np.isfinite(r["dw"]).all()
    assert np.all(r["dw"][7] == 0) and r["db"][7] == 0


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("d", [24, 200])
def test_xent_biases_of_the_lowest_value(ctx, kind, d):
    """A mask of the type's lowest value: as good as closed beside other classes."""
    rng, h, w, y = _problem(14, 33, d, 90)
    bias = np.zeros(90, np.float32)
    bias[::3] = np.finfo(np.float32).min
    y = (y // 3 * 3 + 1).astype(np.int32)
    x = D.Xent(ctx, h, w, y, kind, bias)
    x.grad()
    D.check(x.results(), D.xent_reference(h, w, y, kind, bias))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("d", [24, 200])
def test_xent_nan_stays_in_its_row(ctx, kind, d):
    _, h, w, y = _problem(15, 140, d, 60)
    want = D.xent_reference(h, w, y, kind)
    h[77, 3] = np.nan
    x = D.Xent(ctx, h, w, y, kind)
    x.grad()
    r = x.results()
    assert np.isnan(r["loss"][77]) and np.isnan(r["dh"][77]).all() and np.isnan(r["dw"]).all()
    keep = np.arange(140) != 77
    for name in ("loss", "lse", "dh"):
        r[name], want[name] = r[name][keep], tuple(t[keep] for t in want[name])
    D.check(r, want, ("loss", "lse", "dh"))


@pytest.mark.parametrize("d", [30, 260])
@pytest.mark.parametrize("big", [1e-30, 1e-6, 1.0, 1e6, 1e18])
def test_xent_f32_of_any_magnitude(ctx, big, d):
    """h and w of reciprocal magnitudes: the scores are ordinary, the operands are not."""
    _, h, w, y = _problem(16, 100, d, 150)
    h = (h * np.float32(big)).astype(np.float32)
    w = (w / np.float32(big)).astype(np.float32)
    x = D.Xent(ctx, h, w, y, "f32")
    x.grad()
    D.check(x.results(), D.xent_reference(h, w, y, "f32"))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("d", [30, 260])
def test_xent_large_scores(ctx, kind, d):
    """Scores in the hundreds: one class has nearly all of a row's probability."""
    _, h, w, y = _problem(17, 90, d, 200, scale=120.0)
    x = D.Xent(ctx, h, w, y, kind)
    x.grad()
    D.check(x.results(), D.xent_reference(h, w, y, kind))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("d", [20, 140])
def test_xent_outputs_not_asked_for(ctx, kind, d):
    rng, h, w, y = _problem(18, 60, d, 100)
    full = D.Xent(ctx, h, w, y, kind)
    full.grad()
    want = full.results()
    for ask in ((True, False, False), (False, True, False), (False, False, True),
                (False, False, False)):
        x = D.Xent(ctx, h, w, y, kind)
        x.grad(*ask)
        got = x.results()
        for name, asked in zip(("dh", "dw", "db"), ask):
            assert np.array_equal(got[name], want[name]) if asked else np.all(got[name] == 7.0)
        assert np.array_equal(got["loss"], want["loss"])


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_xent_no_rows(ctx, kind):
    _, h, w, y = _problem(19, 0, 9, 12)
    x = D.Xent(ctx, np.zeros((0, 9), np.float32), w, [0], kind, w_pad=2)
    x.forward()
    x.grad()
    ctx.sync()
    assert np.all(x._matrix(x.dw, 12, 2) == 0)
    assert np.all(ctx.download(x.db, 12, np.float32) == 0)
    assert ctx.download(x.loss, 1, np.float32)[0] == 7.0


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("d", [37, 272])
def test_xent_repeats_bit_for_bit(ctx, kind, d):
    rng, h, w, y = _problem(20, 1500, d, 2100)
    bias = rng.standard_normal(2100).astype(np.float32)
    runs = []
    for _ in range(3):
        x = D.Xent(ctx, h, w, y, kind, bias)
        x.grad()
        runs.append(x.results())
    for r in runs[1:]:
        for name in r:
            assert np.array_equal(r[name], runs[0][name]), name


@pytest.mark.parametrize("d", [3, 150])
def test_xent_gradient_against_differences(ctx, d):
    """Central differences of the loss itself, f32: a step of 2^-6 leaves (third
    derivative) / 6 * 2^-12 and the two losses' rounding over 2^-5."""
    rng, h, w, y = _problem(21, 6, d, 9, scale=1.0)
    bias = rng.standard_normal(9).astype(np.float32)
    x = D.Xent(ctx, h, w, y, "f32", bias)
    x.grad()
    r = x.results()
    step = 2.0 ** -6

    def loss(h, w, b):
        z = D.Xent(ctx, h, w, y, "f32", b)
        z.forward()
        return z.results(False)["loss"].astype(np.float64).sum()

    def slope(which, at):
        args = [h.copy(), w.copy(), bias.copy()]
        args[which][at] += np.float32(step)
        up = loss(*args)
        moved = float(args[which][at])
        args = [h.copy(), w.copy(), bias.copy()]
        args[which][at] -= np.float32(step)
        return (up - loss(*args)) / (moved - float(args[which][at]))

    # the third derivative of log-sum-exp along a direction u is at most max|u|^3
    wide = float(max(np.abs(w).max(), np.abs(h).max(), 1.0)) ** 3 * 6
    tol = wide / 6 * step ** 2 + 6 * 8 * (d + 16) * 2.0 ** -24 / step
    for at in ((0, 0), (3, d - 1)):
        assert abs(slope(0, at) - r["dh"][at]) <= tol
        assert abs(slope(1, at) - r["dw"][at]) <= tol
    assert abs(slope(2, 4) - r["db"][4]) <= tol


# ---- rows sorted by expert and back --------------------------------------------------

def _experts(seed, rows, k, experts, dropped=0.1, skew=True):
    rng = np.random.default_rng(seed)
    e = rng.integers(0, experts, (rows, k))
    if skew:
        e = np.minimum(e, rng.integers(0, experts, (rows, k)))
    e = e.astype(np.int32)
    wild = rng.random((rows, k)) < dropped
    e[wild] = rng.choice(np.array([-1, experts, 2 ** 31 - 1, -2 ** 31], np.int64),
                         int(wild.sum())).astype(np.int32)
    return rng, e


@pytest.mark.parametrize("rows,k,experts", [(0, 2, 4), (1, 1, 1), (1, 3, 8192), (63, 1, 2),
                                            (64, 2, 64), (1000, 1, 4), (4097, 3, 65),
                                            (70001, 2, 1000), (300000, 1, 8192), (50000, 8, 3),
                                            (16385, 1, 2048), (16385, 1, 2049), (9000, 2, 2100),
                                            (600001, 1, 5), (1100000, 1, 1500), (263000, 2, 70),
                                            (17000000, 1, 40)])
def test_sort_by_expert(ctx, rows, k, experts):
    _, e = _experts(rows + k, rows, k, experts)
    x = D.Experts(ctx, e, experts)
    x.sort()
    got = x.order()
    for a, b in zip(got, D.sort_reference(e, experts)):
        assert np.array_equal(a, b)


def test_sort_all_dropped_and_all_to_one(ctx):
    for e in (np.full((5000, 2), -1, np.int32), np.full((5000, 2), 6, np.int32)):
        x = D.Experts(ctx, e, 7)
        x.sort()
        for a, b in zip(x.order(), D.sort_reference(e, 7)):
            assert np.array_equal(a, b)


MOVES = [(1, 1, 1, 1), (5, 3, 2, 4), (64, 64, 1, 3), (65, 130, 2, 7), (1000, 10, 1, 4),
         (777, 37, 3, 600), (4100, 100, 1, 20), (300, 513, 8, 5), (130, 2048, 2, 64)]


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("major", ["row", "feature"])
@pytest.mark.parametrize("blocked", [False, True])
@pytest.mark.parametrize("rows,cols,k,experts", MOVES)
def test_gather_combine_and_gradients(ctx, kind, major, blocked, rows, cols, k, experts):
    rng, e = _experts(rows * 3 + cols, rows, k, experts)
    x = D.Experts(ctx, e, experts)
    x.sort()
    offsets, source, slot = D.sort_reference(e, experts)
    kept, slots = int(offsets[-1]), rows * k
    guard = np.float32(7.0)
    dtype = np.uint16 if kind == "bf16" else np.float32
    call = ctx.call
    plan = ctypes.byref(x.plan)
    pad = 5 if cols % 2 else 0
    # gather: bit for bit
    a = D.rounded(rng.standard_normal((rows, cols)).astype(np.float32), kind)
    _, m = D.rows_matrix(ctx, a, kind, major, pad, blocked)
    out = ctx.upload(D.encode(np.full(slots * cols, guard, np.float32), kind))
    call("mbk_expert_gather", plan, ctypes.byref(m), out)
    ctx.sync()
    want = np.full((slots, cols), guard, np.float32)
    want[:kept] = a[source[:kept] // k]
    want = D.to_sorted(want, offsets, blocked)
    got = D.decode(ctx.download(out, slots * cols, dtype), kind)
    assert np.array_equal(got, want)
    # combine: behind the last slot, and for dropped ones, NaN
    y = D.rounded(rng.standard_normal((slots, cols)).astype(np.float32), kind)
    y[kept:] = np.nan
    ydev = ctx.upload(D.encode(D.to_sorted(y, offsets, blocked), kind))
    weights = rng.standard_normal((rows, k)).astype(np.float32)
    weights[slot < 0] = np.nan
    wdev = ctx.upload(weights)
    terms = np.where(slot[..., None] >= 0, y[slot].astype(np.float64), 0.0)
    wt = np.where(slot >= 0, weights, 0).astype(np.float64)
    for w, wp in ((wt, wdev), (np.where(slot >= 0, 1.0, 0.0), None)):
        p, m = D.rows_matrix(ctx, np.full((rows, cols), guard, np.float32), kind, major, pad,
                             blocked, guard)
        call("mbk_expert_combine", plan, ydev, D.ptr(wp), ctypes.byref(m))
        ctx.sync()
        got = D.read_rows(ctx, p, rows, cols, kind, major, pad, guard).astype(np.float64)
        want = (terms * w[..., None]).sum(1)
        tol = (np.abs(terms) * np.abs(w)[..., None]).sum(1) * (k + 1) * 2.0 ** -24
        tol += (np.abs(want) + tol) * D.HALF[kind]
        assert np.all(np.abs(got - want) <= tol)
    # gradients
    g = D.rounded(rng.standard_normal((rows, cols)).astype(np.float32), kind)
    _, m = D.rows_matrix(ctx, g, kind, major, pad, blocked)
    dy = ctx.upload(D.encode(np.full(slots * cols, guard, np.float32), kind))
    dw = ctx.upload(np.full((rows, k), guard, np.float32))
    for w, wp in ((np.where(slot >= 0, weights, 0), wdev), (np.ones_like(weights), None)):
        call("mbk_expert_combine_grad", plan, ctypes.byref(m), ydev, D.ptr(wp), dy, dw)
        ctx.sync()
        want = np.full((slots, cols), guard, np.float32)
        rowof = source[:kept] // k
        want[:kept] = D.rounded(w.reshape(-1)[source[:kept], None].astype(np.float32) * g[rowof],
                                kind)
        got = D.from_sorted(D.decode(ctx.download(dy, slots * cols, dtype), kind), offsets, cols,
                            blocked)
        assert np.array_equal(got, want)
        prod = g[:, None, :].astype(np.float64) * terms
        tol = np.abs(prod).sum(2) * (cols + 2) * 2.0 ** -24
        got = ctx.download(dw, (rows, k), np.float32)
        assert np.all(np.abs(got - prod.sum(2)) <= tol)
        assert np.all(got[slot < 0] == 0)


# ---- streams and graphs ---------------------------------------------------------------

class Hip:
    """The HIP runtime the library itself runs on."""

    def __init__(self):
        _core.lib()
        self.l = ctypes.CDLL("libamdhip64.so.7")

    def __call__(self, name, *args):
        rc = getattr(self.l, name)(*args)
        assert rc == 0, (name, rc)


def _chain(ctx, x, plan, m, out):
    x.grad()
    ctx.call("mbk_expert_sort", ctypes.byref(plan))
    ctx.call("mbk_expert_gather", ctypes.byref(plan), ctypes.byref(m), out)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("d", [32, 160])
def test_captured_and_replayed_on_a_callers_stream(kind, d):
    hip = Hip()
    stream = ctypes.c_void_p()
    hip("hipStreamCreate", ctypes.byref(stream))
    ctx = mb.Context(0, stream=stream.value)
    graphs = []
    # two graphs on one context, the second of larger sizes: the scratch of the first
    # is outgrown, and must stay
    for n, v in ((200, 300), (900, 1500)):
        rng, h, w, y = _problem(n, n, d, v)
        _, e = _experts(n, n, 2, 5)
        x = D.Xent(ctx, h, w, y, kind)
        s = D.Experts(ctx, e, 5)
        p, m = D.rows_matrix(ctx, h, kind, "row", 0, False)
        out = ctx.upload(D.encode(np.zeros(n * 2 * d, np.float32), kind))
        _chain(ctx, x, s.plan, m, out)
        want = (x.results(), s.order(), ctx.download(out, n * 2 * d, np.uint16 if kind == "bf16"
                                                     else np.float32))
        graph, run = ctypes.c_void_p(), ctypes.c_void_p()
        hip("hipStreamBeginCapture", stream, 0)
        _chain(ctx, x, s.plan, m, out)
        hip("hipStreamEndCapture", stream, ctypes.byref(graph))
        hip("hipGraphInstantiate", ctypes.byref(run), graph, None, None, ctypes.c_size_t(0))
        graphs.append((x, s, out, n, want, graph, run, h, w, y))
    for _ in range(3):
        for x, s, out, n, want, graph, run, h, w, y in graphs:
            clear = np.zeros(n, np.float32)
            err = ctypes.c_char_p()
            for p in (x.loss, x.lse):
                assert _core.lib().mbk_copy_to_device(ctx.ptr, p, clear.ctypes.data, clear.nbytes,
                                                      ctypes.byref(err)) == 0
            hip("hipGraphLaunch", run, stream)
            got = (x.results(), s.order(), ctx.download(out, n * 2 * d, np.uint16 if kind == "bf16"
                                                        else np.float32))
            for name in want[0]:
                assert np.array_equal(got[0][name], want[0][name]), name
            for a, b in zip(got[1], want[1]):
                assert np.array_equal(a, b)
            assert np.array_equal(got[2], want[2])
    for *_, graph, run, h, w, y in graphs:
        hip("hipGraphExecDestroy", run)
        hip("hipGraphDestroy", graph)
    ctx.close()
    hip("hipStreamDestroy", stream)


def test_growing_scratch_under_capture_is_refused():
    hip = Hip()
    stream = ctypes.c_void_p()
    hip("hipStreamCreate", ctypes.byref(stream))
    ctx = mb.Context(0, stream=stream.value)
    _, h, w, y = _problem(1, 50, 20, 30)
    x = D.Xent(ctx, h, w, y, "f32")
    graph = ctypes.c_void_p()
    hip("hipStreamBeginCapture", stream, 2)
    with pytest.raises(mb.MacBoostError, match="before the capture"):
        x.grad()
    hip("hipStreamEndCapture", stream, ctypes.byref(graph))
    hip("hipGraphDestroy", graph)
    x.grad()
    D.check(x.results(), D.xent_reference(h, w, y, "f32"))
    ctx.close()
    hip("hipStreamDestroy", stream)


# ---- together: a round of boosters behind a gate, for many classes -------------------

def _leaf_forest(rng, trees, cols):
    """Depth-1 trees as mbk_predict_forest takes them."""
    f = {"feature": np.full((trees, 3), -1, np.int32), "threshold": np.zeros((trees, 3), np.float32),
         "flags": np.zeros((trees, 3), np.uint8), "leaf": np.zeros((trees, 3), np.float32)}
    f["feature"][:, 0] = rng.integers(0, cols, trees)
    f["threshold"][:, 0] = rng.random(trees)
    f["leaf"][:, 1:] = rng.standard_normal((trees, 2))
    return f


def _predict_reference(f, x):
    out = np.zeros(x.shape[0], np.float32)
    for t in range(f["feature"].shape[0]):
        left = x[:, f["feature"][t, 0]] <= f["threshold"][t, 0]
        out = (out + np.where(left, f["leaf"][t, 1], f["leaf"][t, 2])).astype(np.float32)
    return out


def test_a_round_of_boosters_behind_a_gate(ctx):
    """Rows to the two best of three boosters, each booster's four outputs for its rows,
    their weighted sum as h, the loss over 50 classes, and back: the gate's gradient
    and each booster's targets, quantised for its next tree."""
    rows, cols, dim, classes, experts, k, trees = 1500, 6, 4, 50, 3, 2, 5
    rng = np.random.default_rng(77)
    x = rng.random((rows, cols)).astype(np.float32)
    gate = np.exp(rng.standard_normal((rows, experts)))
    expert = np.argsort(-gate, axis=1, kind="stable")[:, :k].astype(np.int32)
    gates = np.take_along_axis(gate, expert, 1)
    gates = (gates / gates.sum(1, keepdims=True)).astype(np.float32)
    w = rng.standard_normal((classes, dim)).astype(np.float32)
    y = rng.integers(0, classes, rows).astype(np.int32)
    forests = [[_leaf_forest(rng, trees, cols) for _ in range(dim)] for _ in range(experts)]

    s = D.Experts(ctx, expert, experts)
    s.sort()
    offsets, source, slot = s.order()
    _, xm = D.rows_matrix(ctx, x, "f32", "row", 0, True)
    sorted_x = ctx.alloc(rows * k * cols * 4)
    ctx.call("mbk_expert_gather", ctypes.byref(s.plan), ctypes.byref(xm), sorted_x)
    outputs = ctx.alloc(rows * k * dim * 4)
    for e in range(experts):
        n = int(offsets[e + 1] - offsets[e])
        for j in range(dim):
            f = {key: ctx.upload(v) for key, v in forests[e][j].items()}
            ctx.call("mbk_predict_forest", f["feature"], f["threshold"], f["flags"], f["leaf"],
                     None, trees, 3, sorted_x + int(offsets[e]) * cols * 4, n, 255, 0.0,
                     outputs + (int(offsets[e]) * dim + j * n) * 4)
    h, hm = D.rows_matrix(ctx, np.zeros((rows, dim), np.float32), "f32", "row", 0, True)
    gdev = ctx.upload(gates)
    ctx.call("mbk_expert_combine", ctypes.byref(s.plan), outputs, gdev, ctypes.byref(hm))
    loss = D.Xent(ctx, np.zeros((rows, dim), np.float32), w, y, "f32")
    loss.h = h
    loss.grad()
    dm = _core.MbkExpertMatrix(loss.dh, dim, 1, dim, _core.F32, 1)
    d_out, d_gate = ctx.alloc(rows * k * dim * 4), ctx.alloc(rows * k * 4)
    ctx.call("mbk_expert_combine_grad", ctypes.byref(s.plan), ctypes.byref(dm), outputs, gdev,
             d_out, d_gate)
    got = loss.results()

    # the same from the formulas
    per = np.zeros((rows, k, dim))
    for e in range(experts):
        for j in range(dim):
            values = _predict_reference(forests[e][j], x)
            for c in range(k):
                mine = expert[:, c] == e
                per[mine, c, j] = values[mine]
    h_want = (per * gates[..., None].astype(np.float64)).sum(1)
    h_got = ctx.download(h, (rows, dim), np.float32)
    h_tol = (np.abs(per) * gates[..., None]).sum(1) * (k + 1) * 2.0 ** -24 + np.abs(h_want) * 2 ** -24
    assert np.all(np.abs(h_got - h_want) <= h_tol)
    want = D.xent_reference(h_got, w, y, "f32")
    D.check(got, want)
    d_gate_want = (per * got["dh"][:, None, :].astype(np.float64)).sum(2)
    d_gate_tol = (np.abs(per) * np.abs(got["dh"])[:, None, :]).sum(2) * (dim + 2) * 2.0 ** -24
    assert np.all(np.abs(ctx.download(d_gate, (rows, k), np.float32) - d_gate_want) <= d_gate_tol)
    d_out_host = D.from_sorted(ctx.download(d_out, rows * k * dim, np.float32), offsets, dim, True)
    assert np.array_equal(d_out_host, gates.reshape(-1)[source, None] * got["dh"][source // k])

    # each booster's targets for its next tree
    zeros = ctx.upload(np.zeros(rows * k, np.float32))
    for e in range(experts):
        n = int(offsets[e + 1] - offsets[e])
        for j in range(dim):
            at = (int(offsets[e]) * dim + j * n) * 4
            maxima, entries = ctx.alloc(8), ctx.alloc(n * 8)
            ctx.call("mbk_quantize", 0, 0.0, 0.0, d_out + at, zeros, None, n, maxima, entries)
            ctx.sync()
            g = d_out_host[offsets[e]:offsets[e + 1], j]
            top = ctx.download(maxima, 2, np.float32)
            assert top[0] == np.abs(g).max() and top[1] == 1.0
            words = ctx.download(entries, (n, 2), np.uint32)
            assert np.array_equal(words[:, 0], np.arange(n))
            qg = (words[:, 1].view(np.int32) >> 16).astype(np.float64)
            assert np.all(np.abs(qg - g.astype(np.float64) * 32767 / top[0]) <= 0.5 + 2.0 ** -7)

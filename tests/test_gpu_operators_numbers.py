"""Numbers at the ends of their range in the many-class loss, on either side of 32 rows and of
128 outputs."""
import numpy as np
import pytest

import device_ops as D
from test_gpu_operators import _problem, ctx      # noqa: F401

pytestmark = pytest.mark.gpu

KINDS = pytest.mark.parametrize("kind", ["f32", "bf16"])
FORMS = pytest.mark.parametrize("n,d", [(11, 24), (32, 300), (33, 24), (60, 128), (60, 200)])
LOWEST = np.finfo(np.float32).min
U = 2.0 ** -24


def _biased_reference(h, w, y, kind, bias):
    """The loss and its gradients in 64 bits of scores that are rounded to f32 with their
    bias, and how far each may be off.  A class's score is off by its operands' and its
    sum's half steps and by a step of the rounding with the bias, but where a rounding that
    large goes one way for all classes of a probability, as here, by the dot product's alone:
    a bias beyond 2^31 leaves nothing of a dot product of this size."""
    h, w = D.rounded(h, kind).astype(np.float64), D.rounded(w, kind).astype(np.float64)
    n, d = h.shape
    v = w.shape[0]
    b = np.asarray(bias, np.float32).astype(np.float64)
    huge = np.abs(b) > 2.0 ** 31
    split = 0.0 if kind == "bf16" else 3 * 2.0 ** -22
    products = 1 if kind == "bf16" else 3
    dot = h @ w.T
    z = np.where(huge, b, dot + b)
    ez = (np.abs(h) @ np.abs(w).T) * (split + (products * d + 16) * U) + np.abs(z) * 2 * U
    ez[:, huge] = 0.0
    top = z.max(1, keepdims=True)
    e = np.exp(z - top)
    total = e.sum(1, keepdims=True)
    p = e / total
    rows = np.arange(n)
    # log's sum is off by the mean of its terms' errors and its own f32 sum of v terms
    esum = (p * ez).sum(1) * 1.01 + (v + 32) * U
    lse = top[:, 0] + np.log(total[:, 0])
    elz = esum + 4 * U * np.maximum(1, np.abs(lse))
    loss = (top[:, 0] - z[rows, y]) + np.log(total[:, 0])
    eloss = esum + ez[rows, y] + 4 * U * np.abs(loss) + 4 * U * np.log(v)
    g = p.copy()
    g[rows, y] -= 1
    half = 2.0 ** -11 if kind == "bf16" else 2.0 ** -22
    dist = np.where(p > 0, np.minimum(top - z, 200.0), 0)
    eg = p * (ez + esum[:, None] + (3 * dist + 16) * U) + np.abs(g) * half + 2.0 ** -37
    out = {"lse": (lse, elz), "loss": (loss, eloss)}
    off_h = 2.0 ** -11 if kind == "bf16" else 0.0

    def product(left, right, e_left, terms, off):
        return (e_left @ np.abs(right)
                + (np.abs(left) @ np.abs(right)) * (split + off + (products * terms + 16) * U))

    for name, value, err in (("dh", g @ w, product(g, w, eg, v, 0.0)),
                             ("dw", g.T @ h, product(g.T, h, eg.T, n, off_h)),
                             ("db", g.sum(0), eg.sum(0) + np.abs(g).sum(0) * (n + 4) * U)):
        step = D.HALF[kind] if name != "db" else U
        out[name] = (value, err + (np.abs(value) + err) * step)
    # tolerances that could not pass anything else
    for name in ("dh", "dw"):
        value, tol = out[name]
        assert tol.sum() < 0.1 * np.abs(value).sum(), name
    return out


BIASES = {
    "labels_masked": lambda v: np.where(np.arange(v) % 3 == 0, LOWEST, 0.0),
    "all_lowest": lambda v: np.full(v, LOWEST),
    "one_kept_of_low": lambda v: np.where(np.arange(v) == 4, -2.5e38, LOWEST),
    "all_low_two_kinds": lambda v: np.where(np.arange(v) % 2 == 0, -2.5e38, LOWEST),
    "high": lambda v: np.where(np.arange(v) % 2 == 0, 3e38, 0.0),
    "both_ends": lambda v: np.where(np.arange(v) % 2 == 0, -LOWEST, LOWEST),
    "all_1000": lambda v: np.full(v, 1000.0),
    "all_1e10": lambda v: np.full(v, 1e10),
    "all_-1e10": lambda v: np.full(v, -1e10),
    "all_1e20": lambda v: np.full(v, 1e20),
    "some_-1e5": lambda v: np.where(np.arange(v) % 3 == 0, -1e5, 0.0),
}


@KINDS
@FORMS
@pytest.mark.parametrize("what", ["labels_masked", "all_lowest", "one_kept_of_low",
                                  "all_low_two_kinds", "high", "all_1000", "all_1e10", "all_-1e10",
                                  "all_1e20", "some_-1e5"])
def test_finite_biases(ctx, kind, n, d, what):
    """A class is not offered if its bias is -inf, and only then."""
    _, h, w, y = _problem(n + d + 40, n, d, 90)
    bias = BIASES[what](90).astype(np.float32)
    y[::2] = y[::2] // 3 * 3                          # every second label on a masked class
    x = D.Xent(ctx, h, w, y, kind, bias)
    x.grad()
    got, want = x.results(), _biased_reference(h, w, y, kind, bias)
    D.check(got, want)
    x.forward()
    again = x.results(False)
    for name in ("loss", "lse"):
        assert np.array_equal(got[name], again[name])


@KINDS
@FORMS
def test_biases_of_both_ends(ctx, kind, n, d):
    """A loss beyond f32 is infinite; lse and the gradients are not."""
    _, h, w, y = _problem(n + d + 41, n, d, 90)
    bias = BIASES["both_ends"](90).astype(np.float32)
    x = D.Xent(ctx, h, w, y, kind, bias)
    x.grad()
    got, want = x.results(), _biased_reference(h, w, y, kind, bias)
    beyond = y % 2 == 1
    assert np.all(got["loss"][beyond] == np.inf)
    got["loss"], want["loss"] = got["loss"][~beyond], tuple(t[~beyond] for t in want["loss"])
    D.check(got, want)


@KINDS
@FORMS
@pytest.mark.parametrize("big", [1e35, 2e36])
def test_large_class_vectors(ctx, kind, n, d, big):
    """h and w of reciprocal magnitudes: sums of 90 such w still fit f32."""
    _, h, w, y = _problem(n + d + 42, n, d, 90)
    h = (h / np.float32(big)).astype(np.float32)
    w = (w * np.float32(big)).astype(np.float32)
    x = D.Xent(ctx, h, w, y, kind)
    x.grad()
    want = D.xent_reference(h, w, y, kind)
    assert np.abs(want["dh"][0]).max() < 1e38
    D.check(x.results(), want)


@KINDS
@FORMS
def test_weights_that_are_not_finite(ctx, kind, n, d):
    _, h, w, y = _problem(n + d + 43, n, d, 70)
    weights = np.ones(n, np.float32)
    weights[7] = np.nan
    x = D.Xent(ctx, h, w, y, kind, weights=weights)
    x.grad()
    r = x.results()
    assert np.isnan(r["loss"][7]) and np.isnan(r["dh"][7]).all()
    assert np.isnan(r["dw"]).all() and np.isnan(r["db"]).all()
    keep = np.arange(n) != 7
    want = D.xent_reference(h, w, y, kind)
    for name in ("loss", "lse", "dh"):
        r[name], want[name] = r[name][keep], tuple(t[keep] for t in want[name])
    D.check(r, want, ("loss", "lse", "dh"))
    for value in (np.inf, -np.inf):
        weights[7] = value
        x = D.Xent(ctx, h, w, y, kind, weights=weights)
        x.grad()
        r = x.results()
        assert not np.isfinite(r["loss"][7]) and not np.isfinite(r["dw"][y[7]]).any()


@KINDS
@FORMS
@pytest.mark.parametrize("value", [np.nan, np.inf])
def test_classes_not_offered_beside_a_row_not_finite(ctx, kind, n, d, value):
    """What is not offered has gradients of 0, whatever the rows hold."""
    _, h, w, y = _problem(n + d + 44, n, d, 70)
    bias = np.zeros(70, np.float32)
    bias[::7] = -np.inf
    y = (y // 7 * 7 + 1).astype(np.int32)
    h[3, 5] = value
    x = D.Xent(ctx, h, w, y, kind, bias)
    x.grad()
    r = x.results()
    assert np.all(r["dw"][::7] == 0) and np.all(r["db"][::7] == 0)
    assert not np.isfinite(r["dw"][y[3]]).all()


@KINDS
@FORMS
@pytest.mark.parametrize("k", [16, 24, 32, 40])
@pytest.mark.parametrize("side", ["both", "h", "w"])
def test_columns_of_different_sizes(ctx, kind, n, d, k, side):
    """Every eighth column of h 2^k smaller, of w 2^k larger or smaller, or both, where the
    scores stay as they are: f32 sums of products do not mind."""
    _, h, w, y = _problem(n + d + 45, n, d, 150)
    if side in ("both", "h"):
        h[:, ::8] *= np.float32(2.0 ** -k)
    if side in ("both", "w"):
        w[:, ::8] *= np.float32(2.0 ** (k if side == "both" else -k))
    weights = (np.random.default_rng(k).random(n) + 0.5).astype(np.float32)
    x = D.Xent(ctx, h, w, y, kind, weights=weights)
    x.grad()
    want = D.xent_reference(h, w, y, kind, weights=weights)
    if n > 32 and d <= 128:
        # Columns of w and h are packed times 2^-r and 2^r, r half the difference of their largest
        # exponents, to within 1.  f16 terms of operands below 2^14 are off by 2^-25 where
        # that is more than their 22 bits: at least 2^13 is reached by the largest element of all
        # of w and of each row of h.  What that gives from here on k of 2^33 in f32.
        h64, w64 = (D.rounded(a, kind).astype(np.float64) for a in (h, w))
        a = np.log2(np.abs(w64).max(0))
        b = np.log2((np.abs(h64) / np.abs(h64).max(1, keepdims=True)).max(0))
        r = (a - b) / 2
        off_w = 2.0 ** -36 * 2.0 ** r * (np.abs(w64) * 2.0 ** -r).max()
        off_h = 2.0 ** -36 * 2.0 ** -r * (np.abs(h64) * 2.0 ** r).max(1, keepdims=True)
        z = h64 @ w64.T
        g = np.exp(z - z.max(1, keepdims=True))
        g /= g.sum(1, keepdims=True)
        g[np.arange(n), y] -= 1
        g = np.abs(g) * weights.astype(np.float64)[:, None]
        for name, off in (("dh", g.sum(1, keepdims=True) * off_w), ("dw", g.T @ off_h)):
            want[name] = (want[name][0], want[name][1] + off)
    D.check(x.results(), want)


@KINDS
@FORMS
def test_columns_of_zeros_and_of_one_side(ctx, kind, n, d):
    """A column of w that is all zeros beside large values of h, and the other way round."""
    _, h, w, y = _problem(n + d + 46, n, d, 150)
    h[:, 2] *= np.float32(2.0 ** 60)
    w[:, 2] = 0
    w[:, 9] *= np.float32(2.0 ** 60)
    h[:, 9] = 0
    h[:, 11] = w[:, 11] = 0
    h[4] = 0
    x = D.Xent(ctx, h, w, y, kind)
    x.grad()
    r, want = x.results(), D.xent_reference(h, w, y, kind)
    D.check(r, want)
    x = D.Xent(ctx, np.zeros_like(h), w, y, kind)
    x.grad()
    D.check(x.results(), D.xent_reference(np.zeros_like(h), w, y, kind))
    x = D.Xent(ctx, h, np.zeros_like(w), y, kind)
    x.grad()
    D.check(x.results(), D.xent_reference(h, np.zeros_like(w), y, kind))


@KINDS
@FORMS
def test_weight_times_h_past_f32(ctx, kind, n, d):
    """Where the gradient is small the product with h is not: rows that are nearly certain."""
    _, h, w, y = _problem(n + d + 47, n, d, 80)
    y = np.argmax(h @ w.T, 1).astype(np.int32)
    big = np.arange(n) % 4 == 0
    h[big] *= np.float32(16)
    h = (h * np.float32(2.0 ** 60)).astype(np.float32)
    w = (w * np.float32(2.0 ** -60)).astype(np.float32)
    weights = np.where(big, 1e20, 1e10).astype(np.float32)
    assert (np.abs(h.astype(np.float64)).max(1) * weights)[big].max() > 1e39
    x = D.Xent(ctx, h, w, y, kind, weights=weights)
    x.grad()
    got, want = x.results(), D.xent_reference(h, w, y, kind, weights=weights)
    for name in ("dh", "dw", "db"):
        value, tol = want[name]
        fits = np.abs(value) + tol < 3e38
        assert fits.mean() > 0.9
        off = np.abs(got[name].astype(np.float64) - value)
        assert np.all(off[fits] <= tol[fits]), name


@KINDS
@FORMS
def test_what_is_out_changes_no_bit(ctx, kind, n, d):
    """Neither its values nor its size: no other row, class or column notices."""
    _, h, w, y = _problem(n + d + 48, n, d, 90)
    bias = np.zeros(90, np.float32)
    closed = np.arange(90) % 6 == 0
    bias[closed] = -np.inf
    y = (y // 6 * 6 + 1).astype(np.int32)
    weights = np.ones(n, np.float32)
    y[3], y[4], weights[5] = -1, 90, 0
    out = np.isin(np.arange(n), (3, 4, 5))
    runs = []
    for rows, classes in ((0.0, 0.0), (1e-6, 1e6), (1e15, 1e-20), (3e38, 3e38), (np.nan, np.inf)):
        h[out], w[closed] = rows, classes
        x = D.Xent(ctx, h, w, y, kind, bias, weights)
        x.grad()
        runs.append(x.results())
    for r in runs:
        assert np.array_equal(r["lse"][~out], runs[0]["lse"][~out])
        for name in ("loss", "dh", "dw", "db"):
            assert np.array_equal(r[name], runs[0][name]), name

"""Edges of the operators: the same masks and magnitudes on either side of 32 rows, captured
calls of each form, two contexts at once, many choices a row and many experts."""
import ctypes
import threading

import numpy as np
import pytest

import device_ops as D
import macboost_amd as mb
from macboost_amd import _core
from test_gpu_operators import Hip, _experts, _problem, ctx      # noqa: F401

pytestmark = pytest.mark.gpu

KINDS = pytest.mark.parametrize("kind", ["f32", "bf16"])
# few rows; up to 128 outputs; more
FORMS = pytest.mark.parametrize("n,d", [(11, 24), (11, 300), (60, 24), (60, 200)])


@KINDS
@FORMS
def test_no_class_offered(ctx, kind, n, d):
    _, h, w, y = _problem(n + d, n, d, 70)
    h[3] = np.nan
    x = D.Xent(ctx, h, w, y, kind, np.full(70, -np.inf, np.float32))
    x.grad()
    r = x.results()
    assert np.all(r["lse"][np.arange(n) != 3] == -np.inf)
    for name in ("loss", "dh", "dw", "db"):
        assert np.all(r[name] == 0), name


@KINDS
@FORMS
def test_label_not_offered(ctx, kind, n, d):
    _, h, w, y = _problem(n + d + 1, n, d, 50)
    bias = np.zeros(50, np.float32)
    bias[7] = -np.inf
    y[y == 7] = 8
    keep = np.arange(n) != 4
    want = D.xent_reference(h, w, y, kind, bias)
    # the row's own gradient: all classes' probabilities, and no term of the label
    z = D.rounded(h[4], kind).astype(np.float64) @ D.rounded(w, kind).astype(np.float64).T
    z[7] = -np.inf
    p = np.exp(z - z.max())
    p /= p.sum()
    own = p @ np.where(bias[:, None] == 0, D.rounded(w, kind), 0).astype(np.float64)
    y[4] = 7
    x = D.Xent(ctx, h, w, y, kind, bias)
    x.grad()
    r = x.results()
    assert r["loss"][4] == np.inf
    # p's error is twice its scores' (the operands' 22 bits, f32 sums) and G's 11 bits; its sum is 1
    size = np.abs(h[4]).astype(np.float64) @ np.abs(w).T.astype(np.float64)
    off = 2 * size.max() * (3 * 2.0 ** -22 + (3 * d + 16) * 2.0 ** -24) + 2.0 ** -10
    assert np.all(np.abs(r["dh"][4] - own) <= off * (p @ np.abs(w)) + np.abs(own) * 2.0 ** -8 + 1e-6)
    for name in ("loss", "lse", "dh"):
        r[name], want[name] = r[name][keep], tuple(t[keep] for t in want[name])
    D.check(r, want, ("loss", "lse", "dh"))
    assert np.isfinite(r["dw"]).all()
    assert np.all(r["dw"][7] == 0) and r["db"][7] == 0


@KINDS
@FORMS
def test_biases_of_the_lowest_value(ctx, kind, n, d):
    _, h, w, y = _problem(n + d + 2, n, d, 90)
    bias = np.zeros(90, np.float32)
    bias[::3] = np.finfo(np.float32).min
    y = (y // 3 * 3 + 1).astype(np.int32)
    x = D.Xent(ctx, h, w, y, kind, bias)
    x.grad()
    D.check(x.results(), D.xent_reference(h, w, y, kind, bias))


@KINDS
@FORMS
def test_nan_stays_in_its_row(ctx, kind, n, d):
    _, h, w, y = _problem(n + d + 3, n, d, 60)
    want = D.xent_reference(h, w, y, kind)
    h[7, 3] = np.nan
    x = D.Xent(ctx, h, w, y, kind)
    x.grad()
    r = x.results()
    assert np.isnan(r["loss"][7]) and np.isnan(r["dh"][7]).all() and np.isnan(r["dw"]).all()
    keep = np.arange(n) != 7
    for name in ("loss", "lse", "dh"):
        r[name], want[name] = r[name][keep], tuple(t[keep] for t in want[name])
    D.check(r, want, ("loss", "lse", "dh"))


@FORMS
@pytest.mark.parametrize("big", [1e-30, 1e-6, 1e6, 1e18])
def test_f32_of_any_magnitude(ctx, big, n, d):
    _, h, w, y = _problem(n + d + 4, n, d, 150)
    h = (h * np.float32(big)).astype(np.float32)
    w = (w / np.float32(big)).astype(np.float32)
    x = D.Xent(ctx, h, w, y, "f32")
    x.grad()
    D.check(x.results(), D.xent_reference(h, w, y, "f32"))


@KINDS
@FORMS
def test_large_scores(ctx, kind, n, d):
    _, h, w, y = _problem(n + d + 5, n, d, 200, scale=120.0)
    x = D.Xent(ctx, h, w, y, kind)
    x.grad()
    D.check(x.results(), D.xent_reference(h, w, y, kind))


# split products joined in a captured call, too
@KINDS
@pytest.mark.parametrize("n,d,v", [(9, 40, 500), (32, 300, 5000), (60, 100, 4000), (300, 200, 5000)])
def test_captured_calls_of_each_form(kind, n, d, v):
    hip = Hip()
    stream = ctypes.c_void_p()
    hip("hipStreamCreate", ctypes.byref(stream))
    c = mb.Context(0, stream=stream.value)
    _, h, w, y = _problem(n + v, n, d, v)
    x = D.Xent(c, h, w, y, kind)
    x.grad()
    want = x.results()
    graph, run = ctypes.c_void_p(), ctypes.c_void_p()
    hip("hipStreamBeginCapture", stream, 0)
    x.grad()
    hip("hipStreamEndCapture", stream, ctypes.byref(graph))
    hip("hipGraphInstantiate", ctypes.byref(run), graph, None, None, ctypes.c_size_t(0))
    other = D.Xent(c, h[::-1], w, y[::-1], kind)
    for _ in range(3):
        other.grad()                                # the same scratch, in between
        err, clear = ctypes.c_char_p(), np.zeros(n, np.float32)
        for p in (x.loss, x.lse):
            assert _core.lib().mbk_copy_to_device(c.ptr, p, clear.ctypes.data, clear.nbytes,
                                                    ctypes.byref(err)) == 0
        hip("hipGraphLaunch", run, stream)
        got = x.results()
        for name in want:
            assert np.array_equal(got[name], want[name]), name
    hip("hipGraphExecDestroy", run)
    hip("hipGraphDestroy", graph)
    c.close()
    hip("hipStreamDestroy", stream)


def test_two_contexts_at_once():
    problems = [_problem(s, 400, d, 3000) for s, d in ((1, 60), (2, 250))]
    want, got, failed = [], [[], []], []
    for _, h, w, y in problems:
        c = mb.Context(0)
        x = D.Xent(c, h, w, y, "f32")
        x.grad()
        want.append(x.results())
        c.close()

    def work(i):
        try:
            c = mb.Context(0)
            _, h, w, y = problems[i]
            x = D.Xent(c, h, w, y, "f32")
            for _ in range(20):
                x.grad()
                got[i].append(x.results())
            c.close()
        except Exception as e:                      # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    for i in range(2):
        for r in got[i]:
            for name in want[i]:
                assert np.array_equal(r[name], want[i][name]), name


def test_one_context_from_two_threads():
    c = mb.Context(0)
    calls = []
    for s, n, d, v in ((1, 300, 60, 900), (2, 700, 250, 3000)):          # the second outgrows the first
        _, h, w, y = _problem(s, n, d, v)
        calls.append((D.Xent(c, h, w, y, "f32"), D.xent_reference(h, w, y, "f32")))
    failed = []

    def work(x):
        try:
            for _ in range(30):
                x.grad()
        except Exception as e:                      # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(x,)) for x, _ in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    for x, want in calls:
        D.check(x.results(), want)
    c.close()


@KINDS
@pytest.mark.parametrize("major", ["row", "feature"])
@pytest.mark.parametrize("blocked", [False, True])
@pytest.mark.parametrize("rows,cols,k,experts", [(70, 20, 33, 9), (1, 3, 5000, 4), (500, 12, 2, 8192),
                                                 (40000, 1, 1, 3000), (900, 6, 17, 1)])
def test_many_choices_and_experts(ctx, kind, major, blocked, rows, cols, k, experts):
    rng, e = _experts(rows + cols, rows, k, experts)
    x = D.Experts(ctx, e, experts)
    x.sort()
    offsets, source, slot = D.sort_reference(e, experts)
    for a, b in zip(x.order(), (offsets, source, slot)):
        assert np.array_equal(a, b)
    kept, slots = int(offsets[-1]), rows * k
    dtype = np.uint16 if kind == "bf16" else np.float32
    a = D.rounded(rng.standard_normal((rows, cols)).astype(np.float32), kind)
    _, m = D.rows_matrix(ctx, a, kind, major, 0, blocked)
    out = ctx.upload(D.encode(np.full(slots * cols, 7.0, np.float32), kind))
    ctx.call("mbk_expert_gather", ctypes.byref(x.plan), ctypes.byref(m), out)
    ctx.sync()
    want = np.full((slots, cols), 7.0, np.float32)
    want[:kept] = a[source[:kept] // k]
    got = D.decode(ctx.download(out, slots * cols, dtype), kind)
    assert np.array_equal(got, D.to_sorted(want, offsets, blocked))
    # the sum over its k copies
    p, m = D.rows_matrix(ctx, np.zeros((rows, cols), np.float32), kind, major, 0, blocked, 7.0)
    ctx.call("mbk_expert_combine", ctypes.byref(x.plan), out, None, ctypes.byref(m))
    ctx.sync()
    got = D.read_rows(ctx, p, rows, cols, kind, major, 0, 7.0).astype(np.float64)
    copies = (slot >= 0).sum(1)[:, None]
    exact = a.astype(np.float64) * copies
    assert np.all(np.abs(got - exact) <= np.abs(exact) * ((k + 1) * 2.0 ** -24 + D.HALF[kind]) + 1e-37)


@KINDS
@pytest.mark.parametrize("blocked", [False, True])
@pytest.mark.parametrize("order", ["columns", "rows"])
def test_elements_apart(ctx, kind, blocked, order):
    """Rows' matrices whose elements are three apart in either direction."""
    rows, cols, k, experts = 150, 70, 2, 6
    rng, e = _experts(3, rows, k, experts)
    x = D.Experts(ctx, e, experts)
    x.sort()
    offsets, source, slot = D.sort_reference(e, experts)
    kept, slots = int(offsets[-1]), rows * k
    dtype = np.uint16 if kind == "bf16" else np.float32
    stride = (3 * cols + 4, 3) if order == "columns" else (3, 3 * rows + 4)
    at = np.arange(rows)[:, None] * stride[0] + np.arange(cols)[None, :] * stride[1]
    size = int(at.max()) + 1

    def matrix(values, fill):
        flat = np.full(size, fill, np.float32)
        flat[at] = values
        p = ctx.upload(D.encode(flat, kind))
        return p, _core.MbkExpertMatrix(p, *stride, cols, _core.BF16 if kind == "bf16" else _core.F32,
                                        int(blocked))

    a = D.rounded(rng.standard_normal((rows, cols)).astype(np.float32), kind)
    y = D.rounded(rng.standard_normal((slots, cols)).astype(np.float32), kind)
    weights = rng.standard_normal((rows, k)).astype(np.float32)
    plan, wdev = ctypes.byref(x.plan), ctx.upload(weights)
    out, dy = (ctx.upload(D.encode(np.full(slots * cols, 7.0, np.float32), kind)) for _ in range(2))
    ydev, dw = ctx.upload(D.encode(D.to_sorted(y, offsets, blocked), kind)), ctx.alloc(slots * 4)
    _, m = matrix(a, np.nan)
    back, mback = matrix(np.zeros((rows, cols), np.float32), 7.0)
    ctx.call("mbk_expert_gather", plan, ctypes.byref(m), out)
    ctx.call("mbk_expert_combine", plan, ydev, wdev, ctypes.byref(mback))
    ctx.call("mbk_expert_combine_grad", plan, ctypes.byref(m), ydev, wdev, dy, dw)
    ctx.sync()
    row_of = source[:kept] // k
    for p, rows_of in ((out, a[row_of]),
                       (dy, D.rounded(weights.reshape(-1)[source[:kept], None] * a[row_of], kind))):
        want = np.full((slots, cols), 7.0, np.float32)
        want[:kept] = rows_of
        got = D.decode(ctx.download(p, slots * cols, dtype), kind)
        assert np.array_equal(got, D.to_sorted(want, offsets, blocked))
    flat = D.decode(ctx.download(back, size, dtype), kind)
    terms = np.where(slot[..., None] >= 0, y[slot].astype(np.float64), 0.0)
    exact = (terms * weights[..., None]).sum(1)
    tol = (np.abs(terms) * np.abs(weights)[..., None]).sum(1) * (k + 1) * 2.0 ** -24
    tol += (np.abs(exact) + tol) * D.HALF[kind]
    assert np.all(np.abs(flat[at] - exact) <= tol)
    between = np.ones(size, bool)
    between[at] = False
    assert np.all(flat[between] == 7.0)
    prod = a[:, None, :].astype(np.float64) * terms
    got = ctx.download(dw, (rows, k), np.float32)
    assert np.all(np.abs(got - prod.sum(2)) <= np.abs(prod).sum(2) * (cols + 2) * 2.0 ** -24)

"""The norm of many gradients and clipping on the GPU, against plain 64-bit forms."""
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


# (rows, cols, type, pad, shift) of each gradient
LISTS = [
    [(1, 1, "f32", 0, 0)],
    [(1, 3, "bf16", 0, 1), (5, 7, "f32", 2, 0)],
    [(1003, 37, "f32", 3, 0), (1, 1003, "f32", 0, 0), (300, 37, "bf16", 3, 0), (17, 8, "bf16", 0, 0)],
    [(0, 5, "f32", 0, 0), (5, 0, "bf16", 4, 0), (2, 2, "f32", 0, 0)],
    [(1, 8192, "f32", 0, 0), (1, 8193, "bf16", 0, 0), (3, 8191, "f32", 1, 0), (2, 8200, "bf16", 8, 0)],
    [(2, 20001, "f32", 3, 1), (9000, 1, "bf16", 1, 0), (9000, 1, "f32", 3, 0), (1, 100000, "f32", 0, 3)],
    [(64, 64, "bf16", 0, 0)] * 60 + [(10, 10, "f32", 0, 0)] * 60,
    [(5000, 700, "bf16", 0, 0), (3000, 900, "f32", 0, 0), (1, 70000, "f32", 0, 0)],
    # one workgroup's, and just more
    [(1, 32768, "f32", 0, 0)], [(1, 32769, "f32", 0, 0)], [(1, 32768, "bf16", 0, 1)],
    [(256, 1, "f32", 2, 0)] * 32, [(256, 1, "bf16", 1, 0)] * 16 + [(257, 1, "f32", 1, 0)] * 16,
    [(100, 37, "f32", 3, 1), (100, 37, "bf16", 0, 0), (1, 5, "f32", 0, 0), (0, 3, "f32", 0, 0)],
    [(1, 1, "f32", 0, 0)] * 33, [(1, 1, "bf16", 0, 0)] * 32, [(200, 1023, "f32", 1, 0)],
]


def _make(ctx, rng, sizes, scale=1.0):
    a = [D.rounded((rng.standard_normal((r, c)) * scale).astype(np.float32), t)
         for r, c, t, _, _ in sizes]
    return a, [M.Matrix(ctx, x, t, pad, shift, fill=np.nan)
               for x, (_, _, t, pad, shift) in zip(a, sizes)]


def _entry(g, out):
    return (g.ptr, None if out is None else out.ptr, g.rows, g.cols, g.stride, M.CODE[g.kind])


def _norm(a):
    return np.sqrt(sum((x.astype(np.float64) ** 2).sum() for x in a))


def _clip(ctx, entries, max_norm):
    norm = ctx.upload(np.full(3, M.GUARD, np.float32))
    with_list = ctx.tensors(entries)
    ctx.call("mbk_grad_clip", with_list.ptr, max_norm, norm + 4)
    ctx.sync()
    with_list.close()
    got = ctx.download(norm, 3, np.float32)
    assert got[0] == M.GUARD and got[2] == M.GUARD
    return got[1]


@pytest.mark.parametrize("sizes", LISTS)
@pytest.mark.parametrize("ratio", [0.0, 0.3, 1.5, np.inf])
def test_clip(ctx, sizes, ratio):
    rng = np.random.default_rng(len(sizes))
    a, g = _make(ctx, rng, sizes)
    norm = _norm(a)
    most = float(np.float32(norm * ratio)) if np.isfinite(ratio) else np.inf
    by = most / norm if norm > most else 1.0
    outs = [M.blank(ctx, x.rows, x.cols, x.kind, x.pad, x.shift) for x in g]
    got = _clip(ctx, [_entry(x, o) for x, o in zip(g, outs)], most)
    assert abs(got - norm) <= norm * M.U * (1 + 2.0 ** -20)
    for x, o in zip(a, outs):
        want = x.astype(np.float64) * by
        half = 0.0 if by == 1.0 else M.U + (D.HALF[o.kind] if o.kind == "bf16" else 0.0)
        M.close(o.read(), want, np.abs(want) * half * (1 + 2.0 ** -20) + (0 if by == 1.0 else 1e-44))
    for x, m in zip(a, g):                       # the gradients themselves stay
        assert np.array_equal(D.decode(ctx.download(m.at, m.shift + m.rows * m.stride,
                                                    M.DTYPE[m.kind]), m.kind)[m.shift:].reshape(
            m.rows, m.stride)[:, :m.cols], x)


@pytest.mark.parametrize("sizes", LISTS)
def test_in_place_and_norm_only(ctx, sizes):
    rng = np.random.default_rng(9)
    a, g = _make(ctx, rng, sizes)
    for m in g:
        m.fill = np.nan
    norm = _norm(a)
    assert abs(_clip(ctx, [_entry(x, None) for x in g], 0.5) - norm) <= norm * M.U * 1.001
    # every second in place, the others counted only
    most = float(np.float32(norm * 0.25))
    entries = [_entry(x, x if i % 2 == 0 else None) for i, x in enumerate(g)]
    assert abs(_clip(ctx, entries, most) - norm) <= norm * M.U * 1.001
    by = most / norm
    for i, (x, m) in enumerate(zip(a, g)):
        got = D.decode(ctx.download(m.at, m.shift + m.rows * m.stride, M.DTYPE[m.kind]),
                       m.kind)[m.shift:].reshape(m.rows, m.stride)[:, :m.cols]
        want = x * (by if i % 2 == 0 else 1.0)
        half = (M.U + (D.HALF[m.kind] if m.kind == "bf16" else 0.0)) if i % 2 == 0 else 0.0
        M.close(got, want, np.abs(want) * half * 1.001)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_a_norm_that_is_not_finite_changes_nothing(ctx, bad):
    rng = np.random.default_rng(2)
    a, g = _make(ctx, rng, LISTS[2])
    a[2][7, 7] = bad
    g[2] = M.Matrix(ctx, a[2], "bf16", 3)
    outs = [M.blank(ctx, x.rows, x.cols, x.kind, x.pad, x.shift) for x in g]
    got = _clip(ctx, [_entry(x, o) for x, o in zip(g, outs)], 0.5)
    assert np.isnan(got) if np.isnan(bad) else got == np.inf
    for x, o in zip(a, outs):
        M.close(o.read(), x, 0)


def test_norms_beyond_f32_and_of_tiny_values(ctx):
    a = np.full((3, 1000), 3e38, np.float32)
    g, out = M.Matrix(ctx, a, "f32"), M.blank(ctx, 3, 1000, "f32")
    assert _clip(ctx, [_entry(g, out)], 1.0) == np.inf
    want = a.astype(np.float64) / _norm([a])
    M.close(out.read(), want, want * M.U * 1.001)
    a = np.full((3, 1000), 1e-40, np.float32)
    g, out = M.Matrix(ctx, a, "f32"), M.blank(ctx, 3, 1000, "f32")
    got = _clip(ctx, [_entry(g, out)], 1e-39)
    assert abs(got - _norm([a])) <= 1e-44
    want = a.astype(np.float64) * (np.float64(np.float32(1e-39)) / _norm([a]))
    M.close(out.read(), want, 1e-45)
    # all zeros: a norm of 0, and nothing to scale, with max_norm 0 too
    g, out = M.Matrix(ctx, np.zeros((3, 9), np.float32), "f32"), M.blank(ctx, 3, 9, "f32")
    assert _clip(ctx, [_entry(g, out)], 0.0) == 0
    assert not out.read().any()
    assert _clip(ctx, [], 1.0) == 0


def test_lists_and_their_context(ctx):
    g = M.Matrix(ctx, np.ones((2, 8), np.float32), "f32")
    mine = ctx.tensors([_entry(g, None)])
    norm = ctx.upload(np.zeros(1, np.float32))
    other = mb.Context(0)
    with pytest.raises(mb.MacBoostError, match="not one of the context's"):
        other.call("mbk_grad_clip", mine.ptr, 1.0, norm)
    other.close()
    ctx.call("mbk_grad_clip", mine.ptr, 1.0, norm)
    ctx.sync()
    assert ctx.download(norm, 1, np.float32)[0] == 4
    held = ctypes.c_void_p(mine.ptr.value)
    mine.close()
    with pytest.raises(mb.MacBoostError, match="not one of the context's"):
        ctx.call("mbk_grad_clip", held, 1.0, norm)


def test_repeats_bit_for_bit(ctx):
    rng = np.random.default_rng(4)
    a, g = _make(ctx, rng, LISTS[7])
    outs = [M.blank(ctx, x.rows, x.cols, x.kind, x.pad, x.shift) for x in g]
    first = None
    for _ in range(3):
        got = [_clip(ctx, [_entry(x, o) for x, o in zip(g, outs)], 3.0)] + [o.read() for o in outs]
        if first is not None:
            assert all(np.array_equal(x, y) for x, y in zip(got, first))
        first = got

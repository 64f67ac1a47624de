"""Penalties, biases and masks of scores on the GPU, against a plain 64-bit form."""
import ctypes

import numpy as np
import pytest

import macboost_amd as mb
import model_ops as M
from macboost_amd import _core

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = mb.Context(0)
    yield c
    c.close()


def _adjust(ctx, scores, ids=None, lengths=None, bias=None, allowed=None, rep=1.0, pres=0.0,
            freq=0.0, pad=0, out_pad=0, ids_pad=0, shift=0, in_place=False, mask_pad=0):
    n, v = scores.shape
    m = M.Matrix(ctx, scores, "f32", pad, shift, fill=M.GUARD if in_place else np.nan)
    out = m if in_place else M.blank(ctx, n, v, "f32", out_pad, shift)
    hist = 0 if ids is None else ids.shape[1]
    full = np.full((n, hist + ids_pad), 0, np.int32)
    if hist:
        full[:, :hist] = ids
    idev = ctx.upload(full if full.size else np.zeros(1, np.int32))
    mask, stride = None, 0
    if allowed is not None:
        words = np.zeros((allowed.shape[0], allowed.shape[1] + mask_pad), np.uint32)
        words[:, :allowed.shape[1]] = allowed
        mask = ctx.upload(words)
        stride = words.shape[1] if allowed.shape[0] > 1 else 0
    shape = _core.MbkAdjustShape(n, v, m.stride, out.stride, hist, hist + ids_pad, stride, rep, pres,
                                 freq)
    ctx.call("mbk_adjust", ctypes.byref(shape), m.ptr, idev,
             None if lengths is None else ctx.upload(np.asarray(lengths, np.int32)),
             None if bias is None else ctx.upload(np.asarray(bias, np.float32)), mask, out.ptr)
    ctx.sync()
    return out.read()


def _case(seed, n, v, hist):
    rng = np.random.default_rng(seed)
    scores = (rng.standard_normal((n, v)) * 3).astype(np.float32)
    ids = (rng.random((n, hist)) ** 3 * v).astype(np.int32)
    bad = rng.random((n, hist)) < 0.05
    ids[bad] = rng.choice(np.array([-1, v, 2 ** 31 - 1, -2 ** 31], np.int32), bad.sum())
    lengths = rng.integers(-3, hist + 4, n).astype(np.int32)
    bias = rng.standard_normal(v).astype(np.float32)
    allowed = rng.integers(0, 2 ** 32, (n, -(-v // 32)), dtype=np.uint32)
    return rng, scores, ids, lengths, bias, allowed


@pytest.mark.parametrize("n,v,hist", [(1, 1, 1), (1, 1003, 20), (3, 32, 100), (5, 33, 0), (7, 4096, 50),
                                      (2, 4097, 300), (4, 20000, 2000), (300, 100, 5), (2, 3, 5000),
                                      (1, 70001, 1)])
def test_adjust(ctx, n, v, hist):
    rng, scores, ids, lengths, bias, allowed = _case(n + v, n, v, hist)
    for k, (rep, pres, freq) in enumerate(((1.3, 0.0, 0.0), (0.7, 0.5, 0.1), (1.0, -0.5, 0.0),
                                           (1.0, 0.0, 0.3), (1.0, 0.0, 0.0))):
        ln = lengths if k % 2 else None
        b = bias if k != 1 else None
        mask = (None, allowed, allowed[:1], allowed, None)[k]
        got = _adjust(ctx, scores, ids, ln, b, mask, rep, pres, freq, pad=(0, 4, 3, 0, 1)[k],
                      out_pad=(0, 4, 0, 5, 1)[k], ids_pad=k % 2, shift=(0, 0, 1, 4, 0)[k],
                      mask_pad=k % 3)
        M.close(got, *M.adjust_reference(scores, ids, ln, b, mask if mask is None or n > 1 else
                                         mask[:1], rep, pres, freq))


@pytest.mark.parametrize("v", [100, 9001])
def test_in_place(ctx, v):
    _, scores, ids, lengths, bias, allowed = _case(v, 6, v, 40)
    got = _adjust(ctx, scores, ids, lengths, bias, allowed, 1.2, 0.1, 0.2, pad=3, in_place=True)
    M.close(got, *M.adjust_reference(scores, ids, lengths, bias, allowed, 1.2, 0.1, 0.2))


def test_masked_places_hold_anything_and_rows_may_have_none(ctx):
    _, scores, ids, _, bias, allowed = _case(3, 8, 200, 30)
    on = np.unpackbits(allowed.view(np.uint8), axis=1, bitorder="little")[:, :200].astype(bool)
    dirty = scores.copy()
    off = np.argwhere(~on)
    for i, (r, c) in enumerate(off):
        dirty[r, c] = (np.nan, np.inf, -np.inf, -3.4e38, 3.4e38)[i % 5]
    want = M.adjust_reference(scores, ids, None, bias, allowed, 1.5, 0.2, 0.1)
    M.close(_adjust(ctx, dirty, ids, None, bias, allowed, 1.5, 0.2, 0.1), *want)
    assert np.all(_adjust(ctx, dirty, ids, None, bias, np.zeros_like(allowed), 1.5) == -np.inf)


def test_scores_that_are_not_finite(ctx):
    scores = np.array([[np.inf, -np.inf, np.nan, -3.4028235e38, 3.4028235e38, 0.0, -0.0, 1.0]],
                      np.float32)
    ids = np.arange(8, dtype=np.int32)[None]
    got = _adjust(ctx, scores, ids, rep=2.0, pres=1.0)[0]
    assert got[0] == np.inf and got[1] == -np.inf and np.isnan(got[2]) and got[3] == -np.inf
    assert np.array_equal(got[4:], np.float32([1.70141173e38, -1.0, -1.0, -0.5]))
    # nothing asked for: a copy, bit for bit
    got = _adjust(ctx, scores, ids)
    assert np.array_equal(got.view(np.uint32), scores.view(np.uint32))


def test_no_rows(ctx):
    shape = _core.MbkAdjustShape(0, 5, 5, 5, 0, 0, 0, 1.0, 0.0, 0.0)
    ctx.call("mbk_adjust", ctypes.byref(shape), None, None, None, None, None, None)
    ctx.sync()

"""Scratch that the many-class loss takes."""
import ctypes

import numpy as np
import pytest

import macboost_amd as mb
from macboost_amd import _core
from test_gpu_operators import Hip

pytestmark = pytest.mark.gpu


def _free(hip):
    free, total = ctypes.c_size_t(), ctypes.c_size_t()
    hip("hipMemGetInfo", ctypes.byref(free), ctypes.byref(total))
    return free.value


def test_parts_of_many_rows():
    """Operands packed (0.6 GB), one part of dh (0.6 GB), an eighth more, and no second part."""
    rows, dim, classes = 1_200_000, 128, 20_000
    hip, c = Hip(), mb.Context(0)
    h = c.upload(np.zeros((rows, dim), np.float32))
    w = c.upload(np.zeros((classes, dim), np.float32))
    labels = c.upload(np.zeros(rows, np.int32))
    loss, lse, dh = c.alloc(rows * 4), c.alloc(rows * 4), c.alloc(rows * dim * 4)
    shape = _core.MbkXentShape(rows, classes, dim, _core.F32, dim, dim)
    c.sync()
    before = _free(hip)
    c.call("mbk_xent_grad", ctypes.byref(shape), h, w, None, labels, None, loss, lse, dh, None, None)
    c.sync()
    assert before - _free(hip) < 1.8e9
    got = c.download(lse, rows, np.float32)
    assert np.all(np.abs(got - np.log(classes)) <= (classes + 32) * 2.0 ** -24 + 1e-6)
    assert not c.download(dh, (rows, dim), np.float32).any()
    c.close()


def test_loss_of_many_rows_with_and_without_gradients():
    """Bit for bit, also where the parts' size sets their number."""
    rows, dim, classes = 600_000, 128, 20_000
    rng = np.random.default_rng(4)
    c = mb.Context(0)
    h = c.upload(np.tile(rng.standard_normal((6000, dim)).astype(np.float32), (100, 1)))
    w = c.upload((rng.standard_normal((classes, dim)) / 8).astype(np.float32))
    labels = c.upload(np.tile(rng.integers(0, classes, 6000).astype(np.int32), 100))
    loss, lse, dh = c.alloc(rows * 4), c.alloc(rows * 4), c.alloc(rows * dim * 4)
    shape = _core.MbkXentShape(rows, classes, dim, _core.F32, dim, dim)
    got = []
    for name, more in (("mbk_xent_grad", (dh, None, None)), ("mbk_xent", ())):
        c.call(name, ctypes.byref(shape), h, w, None, labels, None, loss, lse, *more)
        c.sync()
        got.append((c.download(loss, rows, np.float32), c.download(lse, rows, np.float32)))
    assert np.array_equal(got[0][0], got[1][0]) and np.array_equal(got[0][1], got[1][1])
    assert np.isfinite(got[0][0]).all()
    c.close()

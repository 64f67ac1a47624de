"""Category vectors, clipping, 4-bit class vectors and penalties over arrays past 2^31 elements:
few rows far apart, of which only what is used is written and read."""
import ctypes

import numpy as np
import pytest

import device_ops as D
import macboost_amd as mb
import model_ops as M
from macboost_amd import _core

pytestmark = pytest.mark.gpu

FAR = 1 << 30            # elements from row to row: the third row lies past 2^31


@pytest.fixture()
def ctx():
    c = mb.Context(0)
    yield c
    c.close()


def _put(ctx, at, a, kind="f32"):
    a = np.ascontiguousarray(D.encode(a, kind) if kind in ("f32", "bf16") else a)
    err = ctypes.c_char_p()
    assert _core.lib().mbk_copy_to_device(ctx.ptr, at, a.ctypes.data, a.nbytes,
                                          ctypes.byref(err)) == 0


class Far:
    """Rows of cols elements, FAR apart."""

    def __init__(self, ctx, a, kind):
        self.ctx, self.kind, (self.rows, self.cols) = ctx, kind, a.shape
        self.size = M.SIZE[kind]
        self.ptr = ctx.alloc(((self.rows - 1) * FAR + self.cols + 64) * self.size)
        for r in range(self.rows):
            _put(ctx, self.ptr + r * FAR * self.size, np.append(a[r], [M.GUARD] * 64), kind)

    def read(self):
        rows = []
        for r in range(self.rows):
            x = D.decode(self.ctx.download(self.ptr + r * FAR * self.size, self.cols + 64,
                                           M.DTYPE[self.kind]), self.kind)
            assert np.all(x[self.cols:] == M.GUARD), "written behind the row"
            rows.append(x[:self.cols])
        return np.array(rows)


def test_rows_far_apart(ctx):
    rng = np.random.default_rng(1)
    kind, n, dim = "bf16", 4, 40
    table = D.rounded(rng.standard_normal((n, dim)).astype(np.float32), kind)
    ids = np.array([3, 0, 2, 3], np.int32)
    t, idev = Far(ctx, table, kind), ctx.upload(ids)
    out = Far(ctx, np.zeros((n, dim), np.float32), kind)
    shape = M.embed_shape(n, n, dim, kind, FAR, FAR, 0.5)
    ctx.call("mbk_embed", shape, t.ptr, idev, None, out.ptr)
    ctx.sync()
    h = out.read()
    M.close(h, *M.embed_reference(table, ids, None, 0.5, kind))
    # its gradient, h as dout, into the table's memory
    ctx.call("mbk_embed_grad", shape, idev, out.ptr, t.ptr, t.ptr)
    ctx.sync()
    M.close(t.read(), *M.embed_grad_reference(h, ids, n, table, 0.5, kind))
    # clipped in place
    norm = ctx.upload(np.zeros(1, np.float32))
    grads = ctx.tensors([(out.ptr, out.ptr, n, dim, FAR, _core.BF16)])
    want = np.sqrt((h.astype(np.float64) ** 2).sum())
    most = float(np.float32(want / 3))
    ctx.call("mbk_grad_clip", grads.ptr, most, norm)
    ctx.sync()
    assert abs(ctx.download(norm, 1, np.float32)[0] - want) <= want * M.U * 1.001
    M.close(out.read(), h * (most / want), np.abs(h) * (most / want) * (M.U + D.HALF[kind]) * 1.001)
    grads.close()


def test_scores_far_apart(ctx):
    rng = np.random.default_rng(2)
    n, dim, classes = 3, 40, 50
    h = D.rounded(rng.standard_normal((n, dim)).astype(np.float32), "bf16")
    w = D.rounded(rng.standard_normal((3, dim)).astype(np.float32), "bf16")
    shape = _core.MbkFourbitShape(3, dim, 32)
    packed = ctx.alloc(_core.fourbit_bytes(shape))
    wf, hf = Far(ctx, w, "bf16"), Far(ctx, h, "bf16")
    ctx.call("mbk_fourbit_pack", ctypes.byref(shape), _core.BF16, wf.ptr, FAR, packed)
    z = Far(ctx, np.zeros((n, 3), np.float32), "f32")
    ctx.call("mbk_fourbit_scores", ctypes.byref(shape), n, _core.BF16, hf.ptr, FAR, packed, None,
             z.ptr, FAR)
    ctx.sync()
    held = M.values(*M.quantised(w, 32), dim)
    M.close(z.read(), *M.scores_reference(h, held, None, "bf16"))
    # penalties
    scores = rng.standard_normal((n, classes)).astype(np.float32)
    s, out = Far(ctx, scores, "f32"), Far(ctx, np.zeros((n, classes), np.float32), "f32")
    ids = rng.integers(0, classes, (n, 6)).astype(np.int32)
    hist = ctx.alloc(((n - 1) * FAR + 64) * 4)
    for r in range(n):
        _put(ctx, hist + r * FAR * 4, ids[r], "i32")
    allowed = rng.integers(0, 2 ** 32, (n, 2), dtype=np.uint32)
    mask = ctx.alloc(((n - 1) * FAR + 64) * 4)
    for r in range(n):
        _put(ctx, mask + r * FAR * 4, allowed[r], "u32")
    shape = _core.MbkAdjustShape(n, classes, FAR, FAR, 6, FAR, FAR, 1.3, 0.2, 0.1)
    ctx.call("mbk_adjust", ctypes.byref(shape), s.ptr, hist, None, None, mask, out.ptr)
    ctx.sync()
    M.close(out.read(), *M.adjust_reference(scores, ids, None, None, allowed, 1.3, 0.2, 0.1))


def test_one_gradient_past_2_to_31_elements(ctx):
    """A matrix of 2^31 + 1024 ones, made by looking them up, and its norm and scaled form."""
    rows, dim = (1 << 21) + 1, 1024
    one = M.Matrix(ctx, np.ones((1, dim), np.float32), "bf16")
    ids = ctx.upload(np.zeros(rows, np.int32))
    big = ctx.alloc(rows * dim * 2 + 128)
    _put(ctx, big + rows * dim * 2, np.full(64, M.GUARD, np.float32), "bf16")
    ctx.call("mbk_embed", M.embed_shape(rows, 1, dim, "bf16", dim, dim), one.ptr, ids, None, big)
    norm = ctx.upload(np.zeros(1, np.float32))
    grads = ctx.tensors([(big, big, rows, dim, dim, _core.BF16)])
    want = np.sqrt(np.float64(rows) * dim)
    ctx.call("mbk_grad_clip", grads.ptr, float(want / 4), norm)
    ctx.sync()
    assert abs(ctx.download(norm, 1, np.float32)[0] - want) <= want * M.U * 1.001
    for at in (0, (1 << 31) - 512, rows * dim - 1024):
        got = D.from_bf16(ctx.download(big + at * 2, 1024, np.uint16))
        assert np.all(got == 0.25)
    assert np.all(D.from_bf16(ctx.download(big + rows * dim * 2, 64, np.uint16)) == M.GUARD)
    # and as dout: every row to one entry
    shape = M.embed_shape(rows, 1, dim, "bf16", dim, dim)
    b = M.blank(ctx, 1, dim, "bf16")
    ctx.call("mbk_embed_grad", shape, ids, big, None, b.ptr)
    ctx.sync()
    assert np.all(b.read() == D.rounded(np.float32(rows * 0.25), "bf16"))
    grads.close()

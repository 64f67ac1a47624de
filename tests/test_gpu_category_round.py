"""Category vectors, the many-class loss, clipping, class vectors in 4 bits and penalties together:
a training step and the answers after it, eagerly, captured into a graph and from several threads."""
import ctypes
import threading

import numpy as np
import pytest

import device_ops as D
import macboost_amd as mb
import model_ops as M
from macboost_amd import _core
from test_gpu_operators import Hip

pytestmark = pytest.mark.gpu


def _set(ctx, at, a):
    a, err = np.ascontiguousarray(a), ctypes.c_char_p()
    assert _core.lib().mbk_copy_to_device(ctx.ptr, at, a.ctypes.data, a.nbytes,
                                          ctypes.byref(err)) == 0


class Round:
    """h = forests' outputs + the row's category vector; the loss over the classes, the gradients of
    both sets of vectors clipped together; W in 4 bits, its scores of h and their penalties."""

    def __init__(self, ctx, seed, rows, dim, classes, entries, kind="f32"):
        self.ctx, self.kind = ctx, kind
        self.rows, self.dim, self.classes, self.entries = rows, dim, classes, entries
        self.rng = np.random.default_rng(seed)
        rng = self.rng
        self.table = D.rounded(rng.standard_normal((entries, dim)).astype(np.float32), kind)
        self.w = D.rounded((rng.standard_normal((classes, dim)) / np.sqrt(dim)).astype(np.float32),
                           kind)
        self.bias = rng.standard_normal(classes).astype(np.float32)
        self.allowed = rng.integers(0, 2 ** 32, (1, -(-classes // 32)), dtype=np.uint32)
        self.ids = rng.integers(-1, entries, rows).astype(np.int32)
        self.labels = rng.integers(0, classes, rows).astype(np.int32)
        self.history = rng.integers(0, classes, (rows, 7)).astype(np.int32)
        self.forests = M.Matrix(ctx, np.zeros((rows, dim), np.float32), kind)
        self.tdev = M.Matrix(ctx, self.table, kind)
        self.idev = ctx.upload(self.ids)
        self.loss = D.Xent(ctx, np.zeros((rows, dim), np.float32), self.w, self.labels, kind,
                           self.bias)
        self.dtable = M.blank(ctx, entries, dim, kind)
        self.clipped = [M.blank(ctx, classes, dim, kind), M.blank(ctx, 1, classes, "f32"),
                        M.blank(ctx, entries, dim, kind)]
        self.norm = ctx.upload(np.zeros(1, np.float32))
        code = M.CODE[kind]
        self.list = ctx.tensors([
            (self.loss.dw, self.clipped[0].ptr, classes, dim, dim, code),
            (self.loss.db, self.clipped[1].ptr, 1, classes, classes, _core.F32),
            (self.dtable.ptr, self.clipped[2].ptr, entries, dim, dim, code)])
        self.shape = _core.MbkFourbitShape(classes, dim, 32)
        self.packed = ctx.alloc(_core.fourbit_bytes(self.shape))
        self.scores = M.blank(ctx, rows, classes, "f32")
        self.hist, self.mask = ctx.upload(self.history), ctx.upload(self.allowed)
        self.out = M.blank(ctx, rows, classes, "f32")

    def inputs(self):
        f = D.rounded(self.rng.standard_normal((self.rows, self.dim)).astype(np.float32), self.kind)
        _set(self.ctx, self.forests.ptr, D.encode(f, self.kind))
        return f

    def run(self):
        ctx, ref = self.ctx, ctypes.byref
        n, d, v, code = self.rows, self.dim, self.classes, M.CODE[self.kind]
        ctx.call("mbk_embed", M.embed_shape(n, self.entries, d, self.kind, d, d, 0.5), self.tdev.ptr,
                 self.idev, self.forests.ptr, self.loss.h)
        self.loss.grad()
        ctx.call("mbk_embed_grad", M.embed_shape(n, self.entries, d, self.kind, d, d, 0.5), self.idev,
                 self.loss.dh, None, self.dtable.ptr)
        ctx.call("mbk_grad_clip", self.list.ptr, 0.75, self.norm)
        ctx.call("mbk_fourbit_pack", ref(self.shape), code, self.loss.w, d, self.packed)
        ctx.call("mbk_fourbit_scores", ref(self.shape), n, code, self.loss.h, d, self.packed,
                 ctx_bias(self), self.scores.ptr, v)
        shape = _core.MbkAdjustShape(n, v, v, v, 7, 7, 0, 1.2, 0.1, 0.05)
        ctx.call("mbk_adjust", ref(shape), self.scores.ptr, self.hist, None, None, self.mask,
                 self.out.ptr)

    def read(self):
        out = dict(self.loss.results())
        out["h"] = D.decode(self.ctx.download(self.loss.h, (self.rows, self.dim),
                                              M.DTYPE[self.kind]), self.kind)
        out["dtable"] = self.dtable.read()
        out["norm"] = self.ctx.download(self.norm, 1, np.float32)
        for name, m in zip(("cdw", "cdb", "cdt"), self.clipped):
            out[name] = m.read()
        out["scores"], out["out"] = self.scores.read(), self.out.read()
        return out

    def check(self, f):
        """Every step against the 64-bit form of the step on what the step before gave."""
        got = self.read()
        M.close(got["h"], *M.embed_reference(self.table, self.ids, f, 0.5, self.kind))
        D.check(got, D.xent_reference(got["h"], self.w, self.labels, self.kind, self.bias))
        M.close(got["dtable"], *M.embed_grad_reference(got["dh"], self.ids, self.entries, None, 0.5,
                                                       self.kind))
        grads = [got["dw"], got["db"][None], got["dtable"]]
        norm = np.sqrt(sum((g.astype(np.float64) ** 2).sum() for g in grads))
        assert abs(got["norm"][0] - norm) <= norm * M.U * 1.001
        by = min(1.0, 0.75 / norm)
        for g, name in zip(grads, ("cdw", "cdb", "cdt")):
            half = M.U + (0 if name == "cdb" or self.kind == "f32" else D.HALF[self.kind])
            M.close(got[name], g * by, np.abs(g * by) * half * 1.001 + 1e-44)
        held = M.values(*M.quantised(self.w, 32), self.dim)
        M.close(got["scores"], *M.scores_reference(got["h"], held, self.bias, self.kind))
        M.close(got["out"], *M.adjust_reference(got["scores"], self.history, None, None, self.allowed,
                                                1.2, 0.1, 0.05))
        return got


def ctx_bias(r):
    return r.loss.bias


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,dim,classes,entries", [(700, 37, 210, 30), (33, 64, 1000, 500),
                                                      (20000, 16, 100, 3000)])
def test_a_round(kind, rows, dim, classes, entries):
    ctx = mb.Context(0)
    r = Round(ctx, rows, rows, dim, classes, entries, kind)
    f = r.inputs()
    r.run()
    r.check(f)
    r.list.close()
    ctx.close()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_captured_and_replayed(kind):
    hip = Hip()
    stream = ctypes.c_void_p()
    hip("hipStreamCreate", ctypes.byref(stream))
    ctx = mb.Context(0, stream=stream.value)
    graphs = []
    # the second one's scratch outgrows the first one's, which has to stay
    for rows, dim, classes, entries in ((300, 20, 64, 25), (17000, 40, 300, 1500)):
        r = Round(ctx, rows, rows, dim, classes, entries, kind)
        f = r.inputs()
        r.run()
        r.check(f)
        graph, run = ctypes.c_void_p(), ctypes.c_void_p()
        hip("hipStreamBeginCapture", stream, 0)
        r.run()
        hip("hipStreamEndCapture", stream, ctypes.byref(graph))
        hip("hipGraphInstantiate", ctypes.byref(run), graph, None, None, ctypes.c_size_t(0))
        r.list.close()                                   # the graph's copy stays
        graphs.append((r, graph, run))
    for _ in range(3):
        for r, graph, run in graphs:
            f = r.inputs()
            hip("hipGraphLaunch", run, stream)
            first = r.check(f)
            other = r.ctx.tensors([(r.dtable.ptr, None, r.entries, r.dim, r.dim, M.CODE[kind])])
            r.ctx.call("mbk_grad_clip", other.ptr, 1.0, r.norm)       # eager work between replays
            other.close()
            hip("hipGraphLaunch", run, stream)
            again = r.check(f)
            assert all(np.array_equal(first[k], again[k]) for k in first)
    for r, graph, run in graphs:
        hip("hipGraphExecDestroy", run)
        hip("hipGraphDestroy", graph)
    ctx.close()
    hip("hipStreamDestroy", stream)


def test_lists_are_not_made_while_the_stream_is_captured():
    hip = Hip()
    stream = ctypes.c_void_p()
    hip("hipStreamCreate", ctypes.byref(stream))
    ctx = mb.Context(0, stream=stream.value)
    g, norm = M.Matrix(ctx, np.ones((2, 8), np.float32), "f32"), ctx.upload(np.zeros(1, np.float32))
    kept = ctx.tensors([(g.ptr, None, 2, 8, 8, 0)])
    idle = ctx.tensors([(g.ptr, None, 2, 8, 8, 0)])
    ctx.call("mbk_grad_clip", kept.ptr, 1.0, norm)
    graph, run = ctypes.c_void_p(), ctypes.c_void_p()
    hip("hipStreamBeginCapture", stream, 2)
    with pytest.raises(mb.MacBoostError, match="being captured"):
        ctx.tensors([(g.ptr, None, 2, 8, 8, 0)])
    ctx.call("mbk_grad_clip", kept.ptr, 1.0, norm)
    kept.close()
    idle.close()
    hip("hipStreamEndCapture", stream, ctypes.byref(graph))
    hip("hipGraphInstantiate", ctypes.byref(run), graph, None, None, ctypes.c_size_t(0))
    for _ in range(2):
        _set(ctx, norm, np.zeros(1, np.float32))
        hip("hipGraphLaunch", run, stream)
        ctx.sync()
        assert ctx.download(norm, 1, np.float32)[0] == 4
    hip("hipGraphExecDestroy", run)
    hip("hipGraphDestroy", graph)
    ctx.close()
    hip("hipStreamDestroy", stream)


def test_calls_from_several_threads_on_one_context():
    ctx = mb.Context(0)
    rounds = [Round(ctx, 50 + i, 400 * (i + 1), 24, 90, 200 * (i + 1)) for i in range(4)]
    inputs = [r.inputs() for r in rounds]
    for r in rounds:
        r.run()
    want = [r.check(f) for r, f in zip(rounds, inputs)]
    errors = []

    def work(r):
        try:
            for _ in range(20):
                r.run()
        except Exception as e:                           # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(r,)) for r in rounds]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    ctx.sync()
    for r, w in zip(rounds, want):
        got = r.read()
        assert all(np.array_equal(got[k], w[k]) for k in w)
    for r in rounds:
        r.list.close()
    ctx.close()

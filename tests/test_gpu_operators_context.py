"""Contexts on a stream that is being captured."""
import ctypes

import pytest

import device_ops as D
import macboost_amd as mb
from macboost_amd import _core
from test_gpu_operators import Hip, _problem

pytestmark = pytest.mark.gpu


def test_contexts_and_a_capture():
    hip = Hip()
    stream = ctypes.c_void_p()
    hip("hipStreamCreate", ctypes.byref(stream))
    c = mb.Context(0, stream=stream.value)
    _, h, w, y = _problem(3, 40, 20, 30)
    x = D.Xent(c, h, w, y, "f32")
    x.grad()
    c.sync()
    graph, run, nodes = ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_size_t()
    hip("hipStreamBeginCapture", stream, 2)
    with pytest.raises(mb.MacBoostError, match="being captured"):
        mb.Context(0, stream=stream.value)
    x.grad()
    _core.lib().mbk_context_destroy(c.ptr)          # not yet
    hip("hipStreamEndCapture", stream, ctypes.byref(graph))
    hip("hipGraphGetNodes", graph, None, ctypes.byref(nodes))
    assert nodes.value >= 4
    hip("hipGraphInstantiate", ctypes.byref(run), graph, None, None, ctypes.c_size_t(0))
    want = D.xent_reference(h, w, y, "f32")
    for _ in range(3):
        hip("hipGraphLaunch", run, stream)
        D.check(x.results(), want)
        x.forward()
        D.check(x.results(False), want, ("loss", "lse"))
    hip("hipGraphExecDestroy", run)
    hip("hipGraphDestroy", graph)
    c.close()
    hip("hipStreamDestroy", stream)

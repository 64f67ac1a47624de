"""Category vectors, clipping, 4-bit scores and penalties on several contexts at once, each on its
own stream and driven by its own thread."""
import ctypes
import threading

import numpy as np
import pytest

import macboost_amd as mb
from test_gpu_category_round import Round
from test_gpu_operators import Hip

pytestmark = pytest.mark.gpu


def test_contexts_on_streams_of_their_own():
    hip, errors, sets = Hip(), [], []
    for i, (rows, dim, classes, entries) in enumerate(((400, 24, 90, 200), (20000, 16, 300, 3000),
                                                       (6000, 40, 1000, 1100))):
        stream = ctypes.c_void_p()
        hip("hipStreamCreate", ctypes.byref(stream))
        r = Round(mb.Context(0, stream=stream.value), 70 + i, rows, dim, classes, entries,
                  "bf16" if i == 1 else "f32")
        f = r.inputs()
        r.run()
        sets.append((r, r.check(f), stream))

    def work(r):
        try:
            for _ in range(30):
                r.run()
        except Exception as e:                           # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(r,)) for r, _, _ in sets]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for r, want, stream in sets:
        r.ctx.sync()
        got = r.read()
        assert all(np.array_equal(got[k], want[k]) for k in want)
        r.list.close()
        r.ctx.close()
        hip("hipStreamDestroy", stream)

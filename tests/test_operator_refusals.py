"""What the seam's operators refuse: the arguments are checked before the context,
so every refusal shows without a GPU, and nothing is read or written."""
import ctypes

import pytest

import macboost_amd as mb
from macboost_amd import _core

P = 0x1000          # a pointer that no refused call follows


def _call(name, *args):
    err = ctypes.c_char_p()
    if getattr(_core.lib(), name)(None, *args, ctypes.byref(err)) != 0:
        raise mb.MacBoostError(_core._take_error(err))


def _shape(**kw):
    f = {"rows": 4, "classes": 5, "dim": 3, "type": 0, "h_stride": 3, "w_stride": 3, **kw}
    return ctypes.byref(_core.MbkXentShape(*(f[k] for k in ("rows", "classes", "dim", "type",
                                                           "h_stride", "w_stride"))))


@pytest.mark.parametrize("change,msg", [
    ({"rows": -1}, "rows must be in"),
    ({"rows": 2 ** 31}, "rows must be in"),
    ({"classes": 0}, "classes must be in"),
    ({"classes": 2 ** 31}, "classes must be in"),
    ({"dim": 0}, "dim must be in"),
    ({"dim": 2 ** 20 + 1, "h_stride": 2 ** 21, "w_stride": 2 ** 21}, "dim must be in"),
    ({"h_stride": 2}, "h_stride and w_stride"),
    ({"w_stride": 2}, "h_stride and w_stride"),
    ({"type": 2}, "type must be"),
    ({}, "null kernel-seam context"),
])
def test_xent_shapes(change, msg):
    for name, grads in (("mbk_xent", ()), ("mbk_xent_grad", (P, P, P))):
        with pytest.raises(mb.MacBoostError, match=msg):
            _call(name, _shape(**change), P, P, None, P, None, P, P, *grads)


@pytest.mark.parametrize("missing", [0, 1, 3, 5, 6])
def test_xent_null_arrays(missing):
    args = [P, P, None, P, None, P, P]
    args[missing] = None
    with pytest.raises(mb.MacBoostError, match="null argument"):
        _call("mbk_xent", _shape(), *args)


def test_xent_null_shape():
    with pytest.raises(mb.MacBoostError, match="null shape"):
        _call("mbk_xent", None, P, P, None, P, None, P, P)


def _plan(**kw):
    f = {"rows": 4, "k": 2, "experts": 3, "expert": P, "offsets": P, "source": P, "slot": P, **kw}
    return ctypes.byref(_core.MbkExpertPlan(*f.values()))


def _matrix(**kw):
    f = {"data": P, "row_stride": 6, "col_stride": 1, "cols": 6, "type": 0, "blocked": 0, **kw}
    return ctypes.byref(_core.MbkExpertMatrix(*f.values()))


@pytest.mark.parametrize("change,msg", [
    ({"rows": -1}, "rows must be"),
    ({"k": 0}, "rows must be"),
    ({"rows": 2 ** 30, "k": 2}, "rows must be"),
    ({"experts": 0}, "experts must be in 1..8192"),
    ({"experts": 8193}, "experts must be in 1..8192"),
    ({"expert": None}, "null plan array"),
    ({"offsets": None}, "null plan array"),
    ({"source": None}, "null plan array"),
    ({"slot": None}, "null plan array"),
    ({}, "null kernel-seam context"),
])
def test_expert_plans(change, msg):
    for name, args in (("mbk_expert_sort", ()), ("mbk_expert_gather", (_matrix(), P)),
                       ("mbk_expert_combine", (P, None, _matrix())),
                       ("mbk_expert_combine_grad", (_matrix(), P, None, P, P))):
        with pytest.raises(mb.MacBoostError, match=msg):
            _call(name, _plan(**change), *args)


@pytest.mark.parametrize("change,msg", [
    ({"cols": 0}, "cols must be positive"),
    ({"cols": (1 << 30) + 1}, "cols must be at most 2"),
    ({"data": None}, "null matrix data"),
    ({"row_stride": 0}, "row_stride and col_stride"),
    ({"col_stride": -1}, "row_stride and col_stride"),
    ({"row_stride": 5}, "row_stride and col_stride"),
    ({"row_stride": 1, "col_stride": 3}, "row_stride and col_stride"),
    ({"type": 7}, "type must be"),
])
def test_expert_matrices(change, msg):
    for name, args in (("mbk_expert_gather", (_matrix(**change), P)),
                       ("mbk_expert_combine", (P, None, _matrix(**change))),
                       ("mbk_expert_combine_grad", (_matrix(**change), P, None, P, P))):
        with pytest.raises(mb.MacBoostError, match=msg):
            _call(name, _plan(), *args)


def test_expert_null_arrays():
    for name, args in (("mbk_expert_gather", (_matrix(), None)),
                       ("mbk_expert_combine", (None, None, _matrix())),
                       ("mbk_expert_combine_grad", (_matrix(), None, None, P, P)),
                       ("mbk_expert_combine_grad", (_matrix(), P, None, None, P)),
                       ("mbk_expert_combine_grad", (_matrix(), P, None, P, None))):
        with pytest.raises(mb.MacBoostError, match="null argument"):
            _call(name, _plan(), *args)
    with pytest.raises(mb.MacBoostError, match="null plan"):
        _call("mbk_expert_sort", None)
    with pytest.raises(mb.MacBoostError, match="null matrix"):
        _call("mbk_expert_gather", _plan(), None, P)


def test_context_on_a_stream():
    with pytest.raises(mb.MacBoostError, match="device must be >= 0"):
        mb.Context(-1, stream=0)
    with pytest.raises(mb.MacBoostError, match="No HIP GPU available"):
        mb.Context(1 << 20, stream=0)

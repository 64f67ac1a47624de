"""What category vectors, lists of gradients, class vectors in 4 bits and penalties refuse: the
arguments are checked before the context, so every refusal shows without a GPU."""
import ctypes
import math

import pytest

import macboost_amd as mb
from macboost_amd import _core

P = 0x1000          # a pointer that no refused call follows


def _call(name, *args):
    err = ctypes.c_char_p()
    if getattr(_core.lib(), name)(None, *args, ctypes.byref(err)) != 0:
        raise mb.MacBoostError(_core._take_error(err))


def _struct(cls, defaults, change):
    return ctypes.byref(cls(**{**defaults, **change}))


EMBED = {"rows": 4, "entries": 5, "dim": 3, "type": 0, "row_stride": 3, "table_stride": 3,
         "scale": 1.0}


@pytest.mark.parametrize("change,msg", [
    ({"rows": -1}, "rows must be in"), ({"rows": 2 ** 31}, "rows must be in"),
    ({"entries": 0}, "entries must be in"), ({"entries": 2 ** 31}, "entries must be in"),
    ({"dim": 0}, "dim must be in"), ({"dim": 2 ** 20 + 1}, "dim must be in"),
    ({"row_stride": 2}, "row_stride and table_stride"),
    ({"table_stride": 2}, "row_stride and table_stride"),
    ({"row_stride": 2 ** 40 + 1}, "row_stride and table_stride"),
    ({"type": 2}, "type must be"), ({"scale": math.inf}, "scale must be finite"),
    ({"scale": math.nan}, "scale must be finite"), ({}, "null kernel-seam context"),
])
def test_embed_shapes(change, msg):
    for name in ("mbk_embed", "mbk_embed_grad"):
        with pytest.raises(mb.MacBoostError, match=msg):
            _call(name, _struct(_core.MbkEmbedShape, EMBED, change), P, P, None, P)


def test_embed_null_arrays():
    for name in ("mbk_embed", "mbk_embed_grad"):
        for missing in (0, 1, 3):
            args = [P, P, None, P]
            args[missing] = None
            with pytest.raises(mb.MacBoostError, match="null argument"):
                _call(name, _struct(_core.MbkEmbedShape, EMBED, {}), *args)
        with pytest.raises(mb.MacBoostError, match="null shape"):
            _call(name, None, P, P, None, P)


TENSOR = {"grad": P, "out": None, "rows": 2, "cols": 3, "stride": 3, "type": 0}


@pytest.mark.parametrize("change,msg", [
    ({"rows": -1}, "rows and cols must be"), ({"cols": -1}, "rows and cols must be"),
    ({"cols": 2 ** 38 + 1, "stride": 2 ** 39}, "rows and cols must be"),
    ({"stride": 2}, "stride must be in"), ({"stride": 2 ** 40 + 1}, "stride must be in"),
    ({"rows": 2 ** 20, "cols": 2 ** 19, "stride": 2 ** 19}, "at most 2.38 elements together"),
    ({"grad": None}, "null gradient"), ({"type": 3}, "type must be"),
    ({"grad": P + 2}, "multiples of their"), ({"out": P + 1, "type": 1}, "multiples of their"),
    ({}, "null kernel-seam context"), ({"rows": 0, "grad": None}, "null kernel-seam context"),
])
def test_tensors(change, msg):
    out = ctypes.c_void_p()
    good, bad = _core.MbkTensor(**TENSOR), _core.MbkTensor(**{**TENSOR, **change})
    with pytest.raises(mb.MacBoostError, match=msg):
        _call("mbk_tensors_create", (_core.MbkTensor * 2)(good, bad), 2, ctypes.byref(out))
    assert not out.value


Q = 0x9000


@pytest.mark.parametrize("pairs,apart", [
    ([(P, P), (P, P)], False), ([(P, Q), (Q, P)], False), ([(P, Q), (P, Q)], False),
    ([(P, P), (P, Q)], False), ([(P, P), (Q, P)], False), ([(P, P), (P, None)], True),
    ([(P, None), (P, None)], True), ([(P, P), (Q, Q)], True), ([(P, Q), (P, None)], True),
])
def test_a_place_has_one_output(pairs, apart):
    """A gradient may be listed again without an output: it counts twice in the norm."""
    out = ctypes.c_void_p()
    made = [_core.MbkTensor(**{**TENSOR, "grad": g, "out": o}) for g, o in pairs]
    empty = _core.MbkTensor(**{**TENSOR, "out": P, "rows": 0})
    msg = "null kernel-seam context" if apart else "also another gradient"
    with pytest.raises(mb.MacBoostError, match=msg):
        _call("mbk_tensors_create", (_core.MbkTensor * 3)(*made, empty), 3, ctypes.byref(out))


def test_lists_and_norms():
    out = ctypes.c_void_p()
    with pytest.raises(mb.MacBoostError, match="count must be"):
        _call("mbk_tensors_create", None, -1, ctypes.byref(out))
    with pytest.raises(mb.MacBoostError, match="null argument"):
        _call("mbk_tensors_create", None, 1, ctypes.byref(out))
    with pytest.raises(mb.MacBoostError, match="null argument"):
        _call("mbk_tensors_create", None, 0, None)
    for most in (-1.0, math.nan, -math.inf):
        with pytest.raises(mb.MacBoostError, match="max_norm must be"):
            _call("mbk_grad_clip", P, most, P)
    with pytest.raises(mb.MacBoostError, match="null argument"):
        _call("mbk_grad_clip", None, 1.0, P)
    with pytest.raises(mb.MacBoostError, match="null argument"):
        _call("mbk_grad_clip", P, 1.0, None)
    with pytest.raises(mb.MacBoostError, match="null kernel-seam context"):
        _call("mbk_grad_clip", P, math.inf, P)
    _core.lib().mbk_tensors_destroy(None, None)


FOURBIT = {"classes": 20, "dim": 40, "group": 32}


@pytest.mark.parametrize("change,msg", [
    ({"classes": 0}, "classes must be in"), ({"classes": 2 ** 31}, "classes must be in"),
    ({"dim": 0}, "dim must be in"), ({"dim": 2 ** 20 + 1}, "dim must be in"),
    ({"group": 16}, "group must be"), ({"group": 0}, "group must be"),
    ({"group": 48}, "group must be"), ({"group": 256}, "group must be"),
])
def test_fourbit_shapes(change, msg):
    shape = _core.MbkFourbitShape(**{**FOURBIT, **change})
    with pytest.raises(mb.MacBoostError, match=msg):
        _call("mbk_fourbit_pack", ctypes.byref(shape), 0, P, 2 ** 20, P)
    with pytest.raises(mb.MacBoostError, match=msg):
        _call("mbk_fourbit_scores", ctypes.byref(shape), 3, 0, P, 2 ** 20, P, None, P, 2 ** 31)
    assert _core.lib().mbk_fourbit_bytes(ctypes.byref(shape)) == -1
    with pytest.raises(mb.MacBoostError):
        _core.fourbit_bytes(shape)


@pytest.mark.parametrize("args,msg", [
    ((0, P, 39, P), "w_stride must be"), ((0, P, 2 ** 40 + 1, P), "w_stride must be"),
    ((2, P, 40, P), "type must be"), ((0, None, 40, P), "null argument"),
    ((0, P, 40, None), "null argument"), ((0, P, 40, P + 8), "multiple of 16"),
    ((1, P, 40, P), "null kernel-seam context"),
])
def test_fourbit_pack(args, msg):
    with pytest.raises(mb.MacBoostError, match=msg):
        _call("mbk_fourbit_pack", _struct(_core.MbkFourbitShape, FOURBIT, {}), *args)


@pytest.mark.parametrize("args,msg", [
    ((-1, 0, P, 40, P, None, P, 20), "rows must be in"),
    ((2 ** 31, 0, P, 40, P, None, P, 20), "rows must be in"),
    ((3, 0, P, 39, P, None, P, 20), "h_stride must be"),
    ((3, 0, P, 40, P, None, P, 19), "score_stride must be"),
    ((3, 5, P, 40, P, None, P, 20), "type must be"),
    ((3, 0, None, 40, P, None, P, 20), "null argument"),
    ((3, 0, P, 40, None, None, P, 20), "null argument"),
    ((3, 0, P, 40, P, None, None, 20), "null argument"),
    ((3, 0, P, 40, P + 4, None, P, 20), "multiple of 16"),
    ((3, 0, P, 40, P, None, P, 20), "null kernel-seam context"),
])
def test_fourbit_scores(args, msg):
    with pytest.raises(mb.MacBoostError, match=msg):
        _call("mbk_fourbit_scores", _struct(_core.MbkFourbitShape, FOURBIT, {}), *args)
    with pytest.raises(mb.MacBoostError, match="null shape"):
        _call("mbk_fourbit_scores", None, *args)


ADJUST = {"rows": 4, "classes": 50, "score_stride": 50, "out_stride": 50, "history": 6,
          "history_stride": 6, "mask_stride": 2, "repetition": 1.0, "presence": 0.0,
          "frequency": 0.0}


@pytest.mark.parametrize("change,msg", [
    ({"rows": -1}, "rows must be in"), ({"rows": 2 ** 31}, "rows must be in"),
    ({"classes": 0}, "classes must be in"), ({"classes": 2 ** 31}, "classes must be in"),
    ({"rows": 2 ** 20, "classes": 2 ** 21}, "at most 2.40"),
    ({"score_stride": 49}, "score_stride and out_stride"),
    ({"out_stride": 49}, "score_stride and out_stride"),
    ({"out_stride": 2 ** 40 + 1}, "score_stride and out_stride"),
    ({"history": -1}, "history must be"), ({"history": 2 ** 24 + 1}, "history must be"),
    ({"history_stride": 5}, "history_stride must be"), ({"mask_stride": 1}, "mask_stride must be"),
    ({"mask_stride": -2}, "mask_stride must be"),
    ({"repetition": 0.0}, "repetition must be"), ({"repetition": -1.0}, "repetition must be"),
    ({"repetition": math.inf}, "repetition must be"),
    ({"repetition": math.nan}, "repetition must be"),
    ({"presence": math.nan}, "presence and frequency"),
    ({"frequency": math.inf}, "presence and frequency"), ({}, "null kernel-seam context"),
])
def test_adjust_shapes(change, msg):
    with pytest.raises(mb.MacBoostError, match=msg):
        _call("mbk_adjust", _struct(_core.MbkAdjustShape, ADJUST, change), P, P, P, P, P, 2 * P)


def test_adjust_arrays():
    shape = _struct(_core.MbkAdjustShape, ADJUST, {})
    for args in ((None, P, None, None, None, P), (P, None, None, None, None, P),
                 (P, P, None, None, None, None)):
        with pytest.raises(mb.MacBoostError, match="null argument"):
            _call("mbk_adjust", shape, *args)
    with pytest.raises(mb.MacBoostError, match="null shape"):
        _call("mbk_adjust", None, P, P, None, None, None, P)
    with pytest.raises(mb.MacBoostError, match="must have its stride"):
        _call("mbk_adjust", _struct(_core.MbkAdjustShape, ADJUST, {"out_stride": 60}), P, P, None,
              None, None, P)

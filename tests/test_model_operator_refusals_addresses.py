"""Addresses that are no multiple of an array's elements: refused before the context, so that it
shows without a GPU."""
import pytest

import macboost_amd as mb
from macboost_amd import _core
from test_model_operator_refusals import ADJUST, EMBED, FOURBIT, P, _call, _struct

MSG = "multiples of their elements' size"
OTHER = 0x9000


def _refused(name, args, at, by):
    with pytest.raises(mb.MacBoostError, match="null kernel-seam context"):
        _call(name, *args)
    moved = list(args)
    moved[at] += by
    with pytest.raises(mb.MacBoostError, match=MSG):
        _call(name, *moved)


@pytest.mark.parametrize("name", ["mbk_embed", "mbk_embed_grad"])
@pytest.mark.parametrize("kind,by", [(_core.F32, 2), (_core.F32, 1), (_core.BF16, 1)])
def test_category_vectors(name, kind, by):
    shape = _struct(_core.MbkEmbedShape, EMBED, {"type": kind})
    for at in (1, 2, 3, 4):
        _refused(name, (shape, P, P, P, OTHER), at, by)
    # elements of 2 bytes lie at multiples of 2, ids at multiples of 4
    if kind == _core.BF16:
        ids = 2 if name == "mbk_embed" else 1
        args = [shape, P + 2, P + 2, P + 2, OTHER + 2]
        args[ids] = P
        _refused(name, tuple(args), ids, 2)


def test_clipping():
    _refused("mbk_grad_clip", (P, 1.0, P), 2, 2)


def test_class_vectors_in_4_bits():
    shape = _struct(_core.MbkFourbitShape, FOURBIT, {})
    _refused("mbk_fourbit_pack", (shape, 0, P, 40, P), 2, 2)
    _refused("mbk_fourbit_pack", (shape, 1, P + 2, 40, P), 2, 1)
    for kind, by in ((0, 2), (1, 1)):
        _refused("mbk_fourbit_scores", (shape, 3, kind, P, 40, P, P, P, 20), 3, by)
    for at in (6, 7):
        _refused("mbk_fourbit_scores", (shape, 3, 1, P + 2, 40, P, P, P, 20), at, 2)


def test_penalties():
    shape = _struct(_core.MbkAdjustShape, ADJUST, {})
    for at in range(1, 7):
        _refused("mbk_adjust", (shape, P, P, P, P, P, OTHER), at, 2)

"""Strides that the many-class loss refuses, without a GPU."""
import pytest

import macboost_amd as mb
from test_operator_refusals import P, _call, _shape


@pytest.mark.parametrize("change,msg", [
    ({"h_stride": 2 ** 40 + 1}, "h_stride and w_stride must be at most"),
    ({"w_stride": 2 ** 62}, "h_stride and w_stride must be at most"),
    ({"h_stride": 2 ** 40, "w_stride": 2 ** 40}, "null kernel-seam context"),
])
def test_xent_large_strides(change, msg):
    for name, grads in (("mbk_xent", ()), ("mbk_xent_grad", (P, P, P))):
        with pytest.raises(mb.MacBoostError, match=msg):
            _call(name, _shape(**change), P, P, None, P, None, P, P, *grads)

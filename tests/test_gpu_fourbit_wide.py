"""Scores from class vectors in 4 bits of many classes on the GPU: turns of one to eight tiles of
columns, the last one shorter, and scores beyond the caches."""
import numpy as np
import pytest

import macboost_amd as mb
import model_ops as M
from test_gpu_fourbit import _problem

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = mb.Context(0)
    yield c
    c.close()


def _check(ctx, kind, group, rows, dim, classes):
    rng, h, w = _problem(rows + group, rows, dim, classes, kind)
    bias = rng.standard_normal(classes).astype(np.float32)
    bias[rng.random(classes) < 0.1] = -np.inf
    held = M.values(*M.quantised(w, group), dim)
    # rows at odd addresses
    got = M.Fourbit(ctx, w, kind, group).scores(h, bias, pad=3, score_pad=2)
    M.close(got, *M.scores_reference(h, held, bias, kind))


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("tiles", [1, 2, 3, 4, 5, 6, 7, 8])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_turns_of_columns(ctx, kind, tiles, group):
    """25001 classes are 98 workgroups: two turns of `tiles` tiles fill the 256 CUs, one has fewer;
    for one tile, fewer classes."""
    columns = (2 * tiles - 1) * 16 - 15
    if tiles == 1:
        rows, classes = (17 if kind == "f32" else 33), 1003
    else:
        rows, classes = (columns + 1) // 2 if kind == "f32" else columns, 25001
    _check(ctx, kind, group, rows, 200, classes)


@pytest.mark.parametrize("kind,group", [("f32", 32), ("bf16", 64)])
def test_scores_beyond_the_caches(ctx, kind, group):
    """40 MB of them, in rows of 50003 that lie 50005 apart."""
    _check(ctx, kind, group, 201, 777, 50003)

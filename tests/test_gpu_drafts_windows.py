"""Attention of trees in a window whose rows stand anywhere behind the cached keys (include/leafhip.h: positions[t] is at
least length - rows; lh_kv_tree's own never pass the request's last key).

Against the plain 64-bit form (drafts_reference.py), within the bound of test_gpu_kv8.py.
"""
from __future__ import annotations

import numpy as np
import pytest

from tests import kv8_reference as ref
from tests.test_gpu_drafts import check_attention, rt, tree_case  # noqa: F401  (rt: fixture)

pytestmark = pytest.mark.gpu

# (length, rows) each; with two heads a KV head: up to 16 rows of it, up to 32, and more
BATCHES = {"few": [(1020, 8), (700, 3), (90, 8), (450, 1), (8, 8)], "split": [(1020, 16), (700, 9), (90, 15), (450, 2), (16, 16)],
           "rows": [(1020, 20), (700, 40), (90, 30), (450, 9), (64, 64)]}


def standing(c, far):
    """The case with its rows at `far(count)` places behind their request's cached keys."""
    before = np.repeat(c["lengths"] - c["rows"], c["rows"])
    c["positions"] = before + far(len(before))
    return c


@pytest.mark.parametrize("form,block", [(ref.INT8, 16), (ref.E4M3, 128)])
@pytest.mark.parametrize("window", [100, 300])
@pytest.mark.parametrize("batch", BATCHES)
def test_rows_behind_the_last_key(rt, batch, window, form, block):  # noqa: F811
    rng = np.random.default_rng(window + block)
    c = tree_case(rng, BATCHES[batch], 4, 2, 64, block, form)
    # whole steps of 64 cached keys between the last that a row at the end of the rows hides and those that its place hides
    check_attention(rt, standing(c, lambda n: rng.integers(0, window + 300, n)), block, form, window)
    # all rows 200 further than their count, and one that hides every key but itself and its ancestors next to it
    check_attention(rt, standing(c, lambda n: np.full(n, 220)), block, form, window)
    c = standing(c, lambda n: rng.integers(0, 40, n))
    c["positions"][5] += 5000
    got = check_attention(rt, c, block, form, window)
    assert np.isfinite(got).all()


@pytest.mark.parametrize("window", [10, 2 ** 30, 2 ** 31 - 300, 2 ** 31 - 1, 2 ** 31, 2 ** 32 - 1])
@pytest.mark.parametrize("batch", BATCHES)
def test_positions_at_the_end_of_their_type(rt, batch, window):  # noqa: F811
    # a row's own place and its window are exact as far as int32 positions and uint32 windows reach
    rng = np.random.default_rng(61)
    c = tree_case(rng, BATCHES[batch], 4, 2, 64, 32, ref.INT8, reach=20)
    c["positions"] = 2 ** 31 - 1 - rng.integers(0, 60, len(c["positions"]))
    check_attention(rt, c, 32, ref.INT8, window)
    c["positions"][::3] = 2 ** 30 + rng.integers(-30, 30, len(c["positions"][::3]))
    check_attention(rt, c, 32, ref.INT8, window)

"""lh_attention_kv8 of scores far from zero, 2^20 to 2^120 and their negatives, against 64 bits (kv8_reference.py).

Queries have one value that is not zero and key scales are powers of two, so that a row's scores are multiples of one
number that no rounding tells apart: keys of the largest score share the weight, all others' is zero (a query value of
2^20 puts them 2^7 apart at least: codes differ by 2^-9, scales by 2^2, the root of the dim is at most 2^4).  What is
left of the bound is its part without scores.
"""
from __future__ import annotations

import numpy as np
import pytest

from tests import kv8_reference as ref
from tests import test_gpu_kv8 as kv8

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rt():
    from leaf_amd import runtime
    runtime.library()
    return runtime


def signed(codes, form, sign):
    """The codes' magnitudes (from 1 or 2^-3 up) with one sign; NaN stays NaN."""
    if form == ref.INT8:
        return np.clip(sign * np.maximum(np.abs(codes.view(np.int8).astype(int)), 1), -127, 127).astype(np.int8).view(np.uint8)
    return np.maximum(codes & 0x7F, 0x20) | np.uint8(0x80 if sign < 0 else 0)


@pytest.mark.parametrize("form", [ref.INT8, ref.E4M3])
@pytest.mark.parametrize("sign", [0, 1, -1])
@pytest.mark.parametrize("size", [2.0 ** 20, 3.0 * 2 ** 24, 1.7 * 2 ** 33, 2.0 ** 70, 1.3 * 2 ** 110])
@pytest.mark.parametrize("batch,heads,kv,dim,block,window", [("ragged", 8, 2, 64, 16, 0), ("mixed", 4, 2, 64, 32, 50), ("chunk", 4, 1, 128, 64, 0),
                                                             ("one key", 2, 1, 80, 16, 0), ("long", 4, 2, 256, 128, 0)])
def test_far_scores(rt, form, sign, size, batch, heads, kv, dim, block, window):
    rng = np.random.default_rng(dim + len(batch))
    c = kv8.attention_case(rng, kv8.BATCHES[batch], heads, kv, dim, block, form)
    if sign:
        c["keys"] = signed(c["keys"], form, sign)
    c["key_scales"] = np.exp2(rng.integers(-2, 1, c["key_scales"].shape)).astype(np.float32)
    c["value_scales"] = np.exp2(rng.integers(-30, 20, c["value_scales"].shape)).astype(np.float32)
    tokens = c["q"].shape[1]
    c["q"][:] = 0.0
    at = rng.integers(0, dim, (heads, tokens))
    signs = np.ones((heads, tokens, 1)) if sign else rng.choice([-1.0, 1.0], (heads, tokens, 1))
    np.put_along_axis(c["q"], at[..., None], (size * signs).astype(np.float32), 2)
    got = kv8.attend_on_gpu(rt, c, block, form, window)
    want = np.full(got.shape, 7.0)
    ref.attention(**c, block=block, form=form, window=window, out=want)
    largest = np.nanmax(np.abs(ref.decode(c["values"], form)).max((2, 3)) * c["value_scales"])
    err = np.abs(got - want).max()
    assert np.isfinite(got).all() and err <= kv8.bound(0.0, c["lengths"].max(), largest), (err, largest)


def test_scores_past_the_largest_number(rt):
    # infinite scores are no numbers; the other rows keep theirs
    c = kv8.attention_case(np.random.default_rng(1), [(40, 1), (300, 1)], 4, 2, 64, 16, ref.INT8)
    c["q"][1, 0] = 3e38
    c["keys"] = signed(c["keys"], ref.INT8, -1)
    got = kv8.attend_on_gpu(rt, c, 16, ref.INT8)
    assert np.isnan(got[0, 1]).all() and np.isfinite(np.delete(got.reshape(-1, 64), 1, 0)).all()

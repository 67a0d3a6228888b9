"""lh_attention_kv8 over blocks whose value scales are up to 2^140 apart, against 64 bits (kv8_reference.py).

A key's weight belongs to the sum of weights whatever its values' scale is: a block of zeros (INT8 scale 1e-12, E4M3
2^-40) beside one of values near 2^107 takes its share of the average.  The bound is test_gpu_kv8.py's, with the
largest value that a row sees; weights below 2^-126 of a row's largest may be lost, which it covers.
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


def largest_seen(c, block, form, window):
    """[tokens, heads]: the largest magnitude among the values that a row sees."""
    heads, tokens, dim = c["q"].shape
    kv = c["keys"].shape[1]
    out = np.zeros((tokens, heads))
    for r, (start, rows, length) in enumerate(zip(c["starts"], c["rows"], c["lengths"])):
        pages = c["table"][r, :-(-length // block)]
        v = np.abs(ref.decode(c["values"][pages], form)).max(2) * c["value_scales"][pages][..., None].astype(np.float64)
        v = v.transpose(1, 0, 2).reshape(kv, -1)                   # [kv, key]
        for i in range(rows):
            last = length - rows + i
            seen = v[:, max(0, last + 1 - window) if window else 0:last + 1].max(1)
            out[start + i] = np.repeat(seen, heads // kv)
    return out


def check(rt, c, block, form, window=0):
    got = kv8.attend_on_gpu(rt, c, block, form, window)
    want = np.full(got.shape, 7.0)
    A = ref.attention(**c, block=block, form=form, window=window, out=want)
    err, limit = np.abs(got - want).max(-1), kv8.bound(A, c["lengths"].max(), largest_seen(c, block, form, window))
    assert np.isfinite(got).all() and (err <= limit).all(), (np.nanmax(err / np.maximum(limit, 1e-300)), np.argwhere(~(err <= limit))[:5])


@pytest.mark.parametrize("form", [ref.INT8, ref.E4M3])
@pytest.mark.parametrize("length,rows", [(32, 1), (32, 2), (33, 33), (64, 20)])
@pytest.mark.parametrize("zeros_first", [False, True])
def test_zeros_keep_their_weight(rt, form, length, rows, zeros_first):
    # equal scores: the output is the mean
    c = kv8.attention_case(np.random.default_rng(1), [(length, rows)], 4, 2, 64, 16, form)
    c["q"][:] = 0.0
    zeros = c["table"][0, zeros_first ^ 1:-(-length // 16):2]
    c["value_scales"][:] = 2.0 ** 100
    c["value_scales"][zeros] = 2.0 ** -40 if form == ref.E4M3 else 1e-12
    c["values"][zeros] = 0
    check(rt, c, 16, form)


@pytest.mark.parametrize("form", [ref.INT8, ref.E4M3])
@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("batch", ["one", "long", "ragged", "few rows", "prompt", "chunk", "mixed", "long chunk"])
@pytest.mark.parametrize("heads,kv,dim,block", [(8, 2, 64, 16), (4, 1, 128, 64), (2, 1, 144, 32)])
def test_scales_at_the_ends(rt, form, window, batch, heads, kv, dim, block):
    # each block at one of both ends or between, in any order; parted tiles among them
    rng = np.random.default_rng(len(batch) + dim)
    c = kv8.attention_case(rng, kv8.BATCHES[batch], heads, kv, dim, block, form)
    c["value_scales"] = np.exp2(rng.choice([-40.0, -39.0, 0.0, 30.0, 99.0, 100.0], c["value_scales"].shape)).astype(np.float32)
    check(rt, c, block, form, window)


@pytest.mark.parametrize("batch", ["ragged", "mixed", "long chunk"])
@pytest.mark.parametrize("rising", [False, True])
def test_scales_that_rise_or_fall(rt, batch, rising):
    # every block's scale is past the one before it, by 2^140 in all: rescales in each step
    rng = np.random.default_rng(3)
    c = kv8.attention_case(rng, kv8.BATCHES[batch], 4, 2, 64, 16, ref.INT8)
    for r, n in enumerate(c["lengths"]):
        pages = c["table"][r, :-(-n // 16)]
        exponents = np.round(np.linspace(-40, 100, len(pages)))
        c["value_scales"][pages] = np.exp2(exponents if rising else exponents[::-1]).astype(np.float32)[:, None]
    check(rt, c, 16, ref.INT8)


@pytest.mark.parametrize("batch", ["ragged", "mixed"])
@pytest.mark.parametrize("size", [2.0 ** -110, 2.0 ** -60, 2.0 ** 116])
def test_scales_all_small_or_all_large(rt, batch, size):
    c = kv8.attention_case(np.random.default_rng(4), kv8.BATCHES[batch], 4, 2, 64, 16, ref.INT8)
    c["value_scales"] = (c["value_scales"] * np.float32(32 * size)).astype(np.float32)
    check(rt, c, 16, ref.INT8)

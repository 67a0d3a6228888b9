"""The 8-bit KV cache on the GPU at sizes whose kernels or routes test_gpu_kv8.py does not reach.

Appends whose waves look at several tokens each, and queries of more values than a workgroup takes at a time; head
dims of three and four partial groups of 64; serving loops whose attention runs in tiles of few rows, or in both kinds.
Compared as there: integers, scales, codes and rotated queries are equal, attention is within its bound.
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


# ------------------------------------------------------------------ append ---
def tokens_a_wave(case):
    """leaf_amd/csrc/rope_kv8.hip: launch_rope_kv8's `each`."""
    slots, kv = case[0], case[2].shape[1]
    return min(max(-(-(len(slots) * 2 * kv // 8) // 512), 1), 8)


RAGGED = [(int(o), int(n)) for o, n in np.random.default_rng(0).integers([0, 1], [16, 41], (120, 2))]
ONES = [(int(o), 1) for o in np.random.default_rng(1).integers(0, 64, 2000)]


@pytest.mark.parametrize("form", [ref.INT8, ref.E4M3])
@pytest.mark.parametrize("each,runs,heads,kv,dim,rotary,block,max_rows", [
    (2, [(0, 2048)], 14, 2, 64, 64, 64, 2048), (3, ONES[:47] + [(7, 500)], 16, 8, 128, 128, 32, 500),
    (8, RAGGED, 8, 8, 32, 32, 16, 40), (8, RAGGED + [(0, 300)], 16, 16, 64, 32, 128, 300), (8, ONES, 8, 8, 16, 8, 64, 1),
    (4, [(3, 1018), (1, 5)], 8, 8, 16, 16, 16, 1018), (8, [(0, 1), (70, 1500), (127, 2), (64, 700)], 8, 8, 48, 36, 128, 1500)])
@pytest.mark.parametrize("gaps", [False, True])
def test_append_of_several_tokens_a_wave(rt, form, each, runs, heads, kv, dim, rotary, block, max_rows, gaps):
    rng = np.random.default_rng(each + dim + form)
    case = kv8.append_case(rng, [(o % block, n) for o, n in runs], heads, kv, dim, rotary, block, form)
    assert tokens_a_wave(case) == each
    slots, positions = case[0], case[1]
    if gaps:                                        # skipped rows, alone and in a row, at each place of a wave's tokens
        skipped = rng.choice(len(slots), len(slots) // 20, replace=False)
        slots[skipped[::2]] = -1
        positions[skipped[1::2]] = 50
        slots[len(slots) // 3:len(slots) // 3 + 11] = -1
    kv8.check_append(rt, case, heads, rotary, block, form, max_rows)


@pytest.mark.parametrize("heads,kv,dim,rotary", [(64, 2, 128, 20), (128, 2, 128, 64), (256, 1, 256, 256), (250, 2, 128, 0), (130, 130, 16, 12)])
def test_append_of_wide_queries(rt, heads, kv, dim, rotary):
    rng = np.random.default_rng(heads)
    case = kv8.append_case(rng, [(3, 1), (0, 19), (15, 2)], heads, kv, dim, rotary, 16, ref.INT8)
    case[0][4] = -1
    kv8.check_append(rt, case, heads, rotary, 16, ref.INT8)


@pytest.mark.parametrize("form", [ref.INT8, ref.E4M3])
@pytest.mark.parametrize("runs", ["decode", "behind", "mixed"])
@pytest.mark.parametrize("dim,rotary,block", [(144, 144, 16), (176, 40, 128), (192, 192, 32), (208, 100, 64), (240, 240, 16)])
def test_append_of_wide_heads(rt, form, runs, dim, rotary, block):
    rng = np.random.default_rng(dim)
    kv8.check_append(rt, kv8.append_case(rng, kv8.RUNS[runs], 4, 2, dim, rotary, block, form), 4, rotary, block, form)


# --------------------------------------------------------------- attention ---
@pytest.mark.parametrize("form", [ref.INT8, ref.E4M3])
@pytest.mark.parametrize("batch", ["one key", "long", "ragged", "few rows", "chunk", "mixed"])
@pytest.mark.parametrize("heads,kv,dim,block,window", [(4, 2, 144, 16, 0), (3, 1, 160, 128, 70), (4, 1, 192, 32, 0), (4, 2, 208, 64, 100),
                                                       (2, 2, 240, 16, 0), (34, 2, 176, 32, 0)])
def test_attention_of_wide_heads(rt, form, batch, heads, kv, dim, block, window):
    rng = np.random.default_rng(dim + len(batch))
    if batch in ("chunk", "mixed") and heads > 8:
        heads = 2 * kv
    kv8.check_attention(rt, kv8.attention_case(rng, kv8.BATCHES[batch], heads, kv, dim, block, form, padding=3), block, form, window)


@pytest.mark.parametrize("form", [ref.INT8, ref.E4M3])
@pytest.mark.parametrize("dim,block", [(144, 32), (208, 16)])
def test_decoding_beside_a_prompt_of_wide_heads(rt, form, dim, block):
    # both kernels in one call, and their parts joined
    rng = np.random.default_rng(dim)
    batch = [(int(rng.integers(1, 300)), 1) for _ in range(30)] + [(170, 60), (2500, 1), (61, 3)]
    kv8.check_attention(rt, kv8.attention_case(rng, batch, 4, 1, dim, block, form, padding=5), block, form)


# ------------------------------------------------------- the three together ---
def few(fresh, most):
    return [[min(n, most) for n in f] for f in fresh]


SINGLE = few([[4, 1, 0, 4, 2, 1], [1, 3, 1, 1, 1, 1], [1, 1, 4, -1, 1, 0], [1, -1, 1, 2, 1, 1]] + 40 * [[1, 1, 1, 1, 1, 1]] +
             [[-1, 1, 1, 1, 1, 4], [3, 1, 1, 1, -1, 1], [1, 1, -1, 1, 4, 1]], 4)
MIXED = [[30, 1, 0, 1, 1, 2, 1, 1], [1, 30, 1, 1, 1, 1, 3, 1], [1, 1, 28, -1, 1, 1, 1, 1], [1, -1, 1, 30, 1, 1, 1, 2]] + \
    12 * [[1] * 8] + [[-1, 1, 1, 1, 1, 1, 1, 25], [33, 1, 1, 1, 1, 1, -1, 1], [17, 1, 1, 1, 1, 1, 17, 1], [1, 1, 1, 4, 4, 4, 1, 1]]
LOOPS = {"few": (SINGLE, (6, 24, 8, 2, 64, 16, 40, 10), 4), "both": (MIXED, (8, 40, 8, 2, 64, 16, 60, 10), 40)}


@pytest.mark.parametrize("form", ["int8", "e4m3"])
@pytest.mark.parametrize("loop", LOOPS)
@pytest.mark.parametrize("captured", [False, True])
def test_serving_loops(rt, form, loop, captured):
    steps, sizes, max_rows = LOOPS[loop]
    device = kv8.Loop(rt, *sizes, form)
    device.pool.batch.max_rows = max_rows
    stream, graphs = rt.Stream(), []

    def step(fresh, qkv, cos, sin):
        device.load(fresh, qkv, cos, sin)
        rt.synchronize()
        if not captured or not graphs:
            device.launch(stream.handle)
            stream.synchronize()
            graphs.append(None)
            return device.results()
        if graphs[0] is None:
            graphs[0] = rt.Graph(stream, lambda: device.launch(stream.handle))
        graphs[0].launch()
        stream.synchronize()
        return device.results()
    kv8.serve(rt, steps, *sizes, rt.KV8_FORMATS[form], step)
    if graphs[0] is not None:
        graphs[0].close()
    stream.close()


@pytest.mark.parametrize("loop", LOOPS)
def test_steps_of_their_own_sizes(rt, loop):
    # a pool of more rows whose batch says each step's own: rows behind them are not touched
    steps, sizes, _ = LOOPS[loop]
    device = kv8.Loop(rt, *sizes, "int8")

    def step(fresh, qkv, cos, sin):
        device.load(fresh, qkv, cos, sin)
        rows = sum(max(n, 0) for n in fresh)
        device.pool.batch.tokens, device.pool.batch.max_rows = rows, max(fresh)
        device.launch()
        out, plan = device.results()
        plan["positions"][rows:] = plan["slots"][rows:] = -1
        return out, plan
    kv8.serve(rt, steps, *sizes, ref.INT8, step)

"""The 8-bit KV cache in blocks on the GPU against plain 64-bit forms (kv8_reference.py).

Integers, scales and codes are equal; rotated queries too (f32 products and sums
of two).  Attention: with A the largest sum of |q||k| of a score, a score is off
by at most 2^-20 A (two f16 parts of a query value leave 2^-22 of the row's
largest, the f32 sums ten roundings of at most A), a weight by that and a few
2^-24, the sums over n keys by n / 16 more roundings; the result by twice a
weight's error times the largest value.
"""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from tests import kv8_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rt():
    from leaf_amd import runtime
    runtime.library()
    return runtime


def ints(rt, a):
    return rt.DeviceArray.of(np.asarray(a, np.int32))


def bound(A, n, values):
    return 2.0 ** -24 * (32 * A + 16 + n / 16) * 2 * values


# ------------------------------------------------------------------ assign ---
def assign_on_gpu(rt, cached, fresh, table, stack, count, block, blocks, tokens, max_rows, aliased=False):
    d = {"cached": ints(rt, cached), "fresh": ints(rt, fresh), "free_blocks": ints(rt, stack), "free_count": ints(rt, [count]),
         "free_left": ints(rt, [-7]), "table": ints(rt, table), "lengths": ints(rt, np.full(len(cached), -7)),
         "starts": ints(rt, np.full(len(cached) + 1, -7)), "rows": ints(rt, np.full(len(cached), -7)),
         "positions": ints(rt, np.full(tokens, -7)), "slots": ints(rt, np.full(tokens, -7))}
    if aliased:
        d["lengths"], d["free_left"] = d["cached"], d["free_count"]
    batch = rt.KvBatch(len(cached), tokens, max_rows, block, blocks, table.shape[1], **{k: v.ptr for k, v in d.items()})
    rt.kv_assign(batch)
    rt.synchronize()
    return {k: d[k].numpy() for k in ("table", "free_blocks", "free_left", "starts", "rows", "lengths", "positions", "slots")}


def held_table(rng, cached, block, width, blocks):
    held = -(-np.asarray(cached) // block)
    order, table, at = rng.permutation(blocks), np.full((len(cached), width), -1), 0
    for r, n in enumerate(held):
        table[r, :n], at = order[at:at + n], at + n
    stack = np.full(blocks, -1)
    stack[:blocks - at] = order[at:]
    return table, stack, blocks - at


@pytest.mark.parametrize("requests,longest,fresh,block,spare,padding,aliased", [
    (1, 0, 1, 16, 4, 0, False), (3, 40, 1, 16, 2, 5, True), (24, 500, 1, 32, 20, 0, True), (65, 300, 200, 64, 90, 77, False),
    (40, 100, 900, 16, 400, 3, True), (1025, 700, 1, 16, 60, 1, False), (4000, 300, 3, 128, 3000, 9, True),
    (7, 90, 5000, 128, 500, 0, False)])
def test_assign(rt, requests, longest, fresh, block, spare, padding, aliased):
    rng = np.random.default_rng(requests + longest)
    cached = rng.integers(0, longest + 1, requests)
    new = rng.integers(0, fresh + 1, requests)             # a request may have none
    new[rng.random(requests) < 0.1] = -1
    held = -(-cached // block)
    width = int(max(held.max(), -(-(cached + new).max() // block))) or 1
    blocks = int(held.sum()) + spare
    table, stack, count = held_table(rng, cached, block, width, blocks)
    tokens = max(1, int(np.maximum(new, 0).sum()) + padding)
    want = ref.assign(cached, new, table, stack, count, block, width, blocks, tokens, max(fresh, 1))
    got = assign_on_gpu(rt, cached, new, table, stack, count, block, blocks, tokens, max(fresh, 1), aliased)
    for name in want:
        assert np.array_equal(got[name], want[name]), name


def test_assign_turns_away(rt):
    # more new tokens than max_rows, than the table has room for, rows past the arrays, a negative length; the pool runs out
    cached, new = np.array([60, 0, 10, 5, 0, 30, 2, -3]), np.array([5, 9, -1, 60, 4, 2, 3, 1])
    table, stack, count = held_table(np.random.default_rng(0), np.maximum(cached, 0), 16, 4, 14)
    for tokens, free, rows in ((90, count, 8), (80, count, 8), (90, 0, 60), (90, 1, 8), (10, count, 9)):
        want = ref.assign(np.maximum(cached, 0), np.where(cached < 0, 10 ** 6, new), table, stack, free, 16, 4, 14, tokens, rows)
        got = assign_on_gpu(rt, cached, new, table, stack, free, 16, 14, tokens, rows)
        for name in ("table", "free_blocks", "free_left", "rows", "lengths"):
            skip = 7 if name == "lengths" else -1
            assert np.array_equal(np.delete(got[name], skip) if skip >= 0 else got[name],
                                  np.delete(want[name], skip) if skip >= 0 else want[name]), (name, tokens, free)
        assert got["lengths"][7] == -3


def test_assign_bad_counts(rt):
    # a free count out of range, more returned than the pool holds, huge numbers: nothing is written out of bounds
    cached, new = np.array([64, 2 ** 31 - 1, 64, 0]), np.array([-1, 2 ** 31 - 1, -1, 2 ** 31 - 1])
    table = np.arange(16).reshape(4, 4)
    for count in (-5, 3, 2 ** 31 - 1):
        got = assign_on_gpu(rt, cached, new, table, np.arange(10), count, 16, 10, 6, 6)
        assert list(got["rows"]) == [0, 0, 0, 0] and (got["slots"] == -1).all() and (got["positions"] == -1).all()
        assert got["free_left"][0] == min(10, max(count, 0) + 8) and list(got["starts"]) == [0, 0, 6, 6, 6]


# ------------------------------------------------------------------ append ---
def tables(rng, positions, half):
    return (rng.standard_normal((positions, max(half, 1))).astype(np.float32) for _ in range(2))


def step_slots(rng, runs, block, blocks):
    """Slots of runs (offset, tokens), each over blocks of its own, and positions."""
    order, at, slots = rng.permutation(blocks), 0, []
    for offset, n in runs:
        places = np.arange(offset, offset + n)
        pages = order[at:at + -(-(offset + n) // block)]
        at += len(pages)
        slots.append(pages[places // block] * block + places % block)
    return np.concatenate(slots)


def rope_on_gpu(rt, slots, positions, keys, values, ks, vs, qkv, heads, rotary, cos, sin, block, form, max_rows, q0):
    blocks, kv, _, dim = keys.shape
    d = {"positions": ints(rt, positions), "slots": ints(rt, slots)}
    dk, dv, dks, dvs, dqkv, dc, ds, dq = (rt.DeviceArray.of(a) for a in (keys, values, ks, vs, qkv, cos, sin, q0))
    batch = rt.KvBatch(requests=1, tokens=len(slots), max_rows=max_rows, block=block, blocks=blocks, width=1,
                       positions=d["positions"].ptr, slots=d["slots"].ptr)
    cache = rt.Kv8(dk.ptr, dv.ptr, dks.ptr, dvs.ptr, kv, dim, form)
    rt.rope_kv8(batch, cache, dqkv, heads, rotary, dc, ds, dq)
    rt.synchronize()
    return dq.numpy(), dk.numpy(), dv.numpy(), dks.numpy(), dvs.numpy()


def append_case(rng, runs, heads, kv, dim, rotary, block, form, spread=1.0, spoil=()):
    slots = step_slots(rng, runs, block, 2 + sum(-(-(o + n) // block) for o, n in runs))
    blocks, tokens = 2 + sum(-(-(o + n) // block) for o, n in runs), len(slots)
    positions = rng.integers(0, 50, tokens)
    qkv = (rng.standard_normal((tokens, heads + 2 * kv, dim)) * np.exp(spread * rng.standard_normal((tokens, 1, 1)))).astype(np.float32)
    keys, values = (rng.integers(0, 255, s, np.uint8) for s in ((blocks, kv, block, dim), (blocks, kv, dim, block)))
    if form == ref.E4M3:
        keys[(keys & 127) == 127] -= 1
        values[(values & 127) == 127] -= 1
    else:
        keys[keys == 128] = 129
        values[values == 128] = 129
    exponents = rng.integers(-9, -2, (2, blocks, kv)).astype(np.float32)
    ks, vs = np.exp2(exponents if form == ref.E4M3 else exponents + rng.random((2, blocks, kv))).astype(np.float32)
    cos, sin = tables(rng, 50, rotary // 2)
    for t, what in spoil:
        qkv[t] = what
    return slots, positions, keys, values, ks, vs, qkv, cos, sin


def check_append(rt, case, heads, rotary, block, form, max_rows=1 << 20):
    slots, positions, keys, values, ks, vs, qkv, cos, sin = case
    tokens, kv, dim = len(slots), keys.shape[1], keys.shape[3]
    q0 = np.full((heads, tokens, dim), 7.0, np.float32)
    got = rope_on_gpu(rt, slots, positions, keys, values, ks, vs, qkv, heads, rotary, cos, sin, block, form, max_rows, q0)
    wk, wv, wks, wvs = keys.copy(), values.copy(), ks.copy(), vs.copy()
    usable = (slots >= 0) & (slots < len(keys) * block) & (positions >= 0) & (positions < len(cos))
    slots = np.where(usable, slots, -1)
    half = rotary // 2
    c, s = cos[np.where(usable, positions, 0)][:, None, :half], sin[np.where(usable, positions, 0)][:, None, :half]
    with np.errstate(all="ignore"):
        turned = ref.rotated(qkv[:, :heads + kv], c, s)
        ref.append(wk, wks, turned[:, heads:], slots, block, form, False)
        ref.append(wv, wvs, qkv[:, heads + kv:], slots, block, form, True)
    want_q = np.where(usable[None, :, None], turned[:, :heads].transpose(1, 0, 2), 7.0)
    assert np.array_equal(got[0], want_q, equal_nan=True)
    for g, w, name in zip(got[1:], (wk, wv, wks, wvs), ("keys", "values", "key scales", "value scales")):
        assert np.array_equal(g, w, equal_nan=g.dtype == np.float32), (name, np.argwhere(g != w)[:4])


# runs (offset in the first block, tokens): decode steps at the start, inside and at the end of a block, prompts that
# begin inside one and end inside another, whole blocks
RUNS = {"decode": [(0, 1), (5, 1), (15, 1), (9, 1), (3, 1)], "prompt": [(0, 67)], "behind": [(11, 150), (0, 16), (15, 2)],
        "mixed": [(3, 1), (0, 40), (1, 1), (14, 35), (7, 3)]}


@pytest.mark.parametrize("form", [ref.INT8, ref.E4M3])
@pytest.mark.parametrize("runs", RUNS)
@pytest.mark.parametrize("heads,kv,dim,rotary,block", [(4, 2, 64, 64, 16), (14, 2, 64, 64, 64), (8, 8, 128, 64, 32),
                                                       (3, 1, 80, 20, 128), (2, 2, 256, 256, 64), (5, 5, 16, 0, 16),
                                                       (6, 3, 48, 36, 32), (32, 1, 112, 112, 128)])
def test_append(rt, form, runs, heads, kv, dim, rotary, block):
    rng = np.random.default_rng(dim + block + form)
    check_append(rt, append_case(rng, RUNS[runs], heads, kv, dim, rotary, block, form), heads, rotary, block, form)


@pytest.mark.parametrize("form", [ref.INT8, ref.E4M3])
def test_append_more_than_64_behind_a_start(rt, form):
    # blocks of 128 that take 64 tokens and more from a slot inside them, the largest value last: one run, one rounding
    rng = np.random.default_rng(11)
    runs = [(1, 127), (37, 91), (63, 65), (64, 64), (5, 64)]
    case = append_case(rng, runs, 4, 2, 64, 64, 128, form)
    case[6][np.cumsum([n for _, n in runs]) - 1] *= np.float32(37.0)
    check_append(rt, case, 4, 64, 128, form)


@pytest.mark.parametrize("form", [ref.INT8, ref.E4M3])
def test_append_extremes(rt, form):
    # zeros, tiny and huge values beside each other; a scale that doubles makes ties of odd codes
    rng = np.random.default_rng(3)
    runs = [(0, 20), (4, 1), (7, 1), (2, 9), (0, 3), (1, 1)]
    case = append_case(rng, runs, 2, 2, 32, 32, 16, form, spread=12.0)
    slots, positions, keys, values, ks, vs, qkv, cos, sin = case
    qkv[20], qkv[22], cos[:], sin[:] = 0.0, 1e-30, 1.0, 0.0
    qkv[21] = 3e38
    qkv[-1] = np.clip(qkv[-1], -1, 1)
    page = slots[-1] // 16
    vs[page] = ks[page] = 0.5 if form == ref.E4M3 else np.float32(100 / 127)
    qkv[-1, :, 0] = 448.0 if form == ref.E4M3 else 200.0
    check_append(rt, case, 2, 32, 16, form)


@pytest.mark.parametrize("form", [ref.INT8, ref.E4M3])
def test_append_borders(rt, form):
    # values next to halfway between two codes
    rng = np.random.default_rng(4)
    case = append_case(rng, [(0, 128)], 1, 1, 64, 0, 128, form)
    qkv = case[6]
    top = np.float32(5.3)
    scale = np.float64(ref.needed_scale(top, form))
    codes = rng.integers(0, 127, (128, 3, 64))
    levels = ref.decode(codes.astype(np.uint8), form)
    next_up = ref.decode(np.minimum(codes + 1, 126 + (form == ref.INT8)).astype(np.uint8), form)
    qkv[:] = ((levels + next_up) / 2 * scale).astype(np.float32)
    for step in range(3):
        qkv[step::4] = np.nextafter(qkv[step::4], np.float32([0, 10, -10][step]))
    qkv = np.minimum(qkv, top)
    qkv[0] = top
    case[6][:] = qkv
    check_append(rt, case, 1, 0, 128, form)


@pytest.mark.parametrize("form", [ref.INT8, ref.E4M3])
@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf])
def test_append_not_finite(rt, form, what):
    rng = np.random.default_rng(5)
    case = append_case(rng, [(0, 5), (3, 1), (0, 40), (9, 2)], 2, 1, 64, 64, 16, form, spoil=[(2, what), (5, what), (20, what)])
    case[4][case[0][46] // 16] = np.nan               # a block that was spoilt before
    check_append(rt, case, 2, 64, 16, form)


@pytest.mark.parametrize("form", [ref.INT8, ref.E4M3])
def test_append_skipped_tokens(rt, form):
    # slots and positions outside the pool and the tables, padding rows at the end and inside
    rng = np.random.default_rng(6)
    case = append_case(rng, [(0, 30), (3, 1), (0, 20), (5, 4)], 4, 2, 64, 64, 16, form)
    slots, positions = case[0], case[1]
    slots[[4, 30, 54]] = [-1, len(case[2]) * 16, 2 ** 31 - 1]
    positions[[9, 40, 41]] = [-1, 50, 2 ** 31 - 1]
    slots[45:50] = -5
    check_append(rt, case, 4, 64, 16, form)


@pytest.mark.parametrize("max_rows", [1, 3])
def test_append_of_few_rows(rt, max_rows):
    rng = np.random.default_rng(7)
    runs = [(int(rng.integers(0, 64)), max_rows) for _ in range(70)]
    check_append(rt, append_case(rng, runs, 8, 2, 128, 128, 64, ref.INT8), 8, 128, 64, ref.INT8, max_rows)


def test_e4m3_conversion_is_the_nearest(rt):
    # every code's neighbourhood: exact values, halfway, just below and above
    levels = ref.E4M3_VALUES[:127]
    half = (levels[:-1] + levels[1:]) / 2
    x = np.concatenate([levels, half, np.nextafter(half.astype(np.float32), np.float32(0)),
                        np.nextafter(half.astype(np.float32), np.float32(500))]).astype(np.float32)
    x = np.concatenate([x, -x])
    x = np.concatenate([x, np.full(-len(x) % 64, 448)]).astype(np.float32)
    x[-1] = 448
    rows = x.reshape(-1, 1, 64)
    tokens = len(rows)
    assert tokens <= 16
    qkv = np.concatenate([np.zeros_like(rows), rows, rows], 1)
    keys, values = np.zeros((1, 1, 16, 64), np.uint8), np.zeros((1, 1, 64, 16), np.uint8)
    case = (np.arange(tokens), np.zeros(tokens, int), keys, values, np.zeros((1, 1), np.float32), np.zeros((1, 1), np.float32), qkv,
            np.ones((1, 1), np.float32), np.zeros((1, 1), np.float32))
    check_append(rt, case, 1, 0, 16, ref.E4M3)


# --------------------------------------------------------------- attention ---
def cache_of(rng, blocks, kv, block, dim, form, spread=0.5):
    keys, values = (ref.encode(np.clip(s[1] * rng.standard_normal(s[0]), -440, 440), form)
                    for s in (((blocks, kv, block, dim), 40), ((blocks, kv, dim, block), 40)))
    ks, vs = (np.exp2(np.round(spread * rng.standard_normal((blocks, kv)) * (1 if form == ref.E4M3 else 64)) / (1 if form == ref.E4M3 else 64) - 5)
              .astype(np.float32) for _ in range(2))
    return keys, values, ks, vs


def attention_case(rng, requests, heads, kv, dim, block, form, padding=0, spread=0.5):
    """requests: (length, rows) each."""
    lengths, rows = (np.array(a) for a in zip(*requests))
    starts = np.concatenate([[0], np.cumsum(rows)])
    held = -(-lengths // block)
    blocks, width = int(held.sum()) + 1, int(held.max()) + 1
    table = np.full((len(rows), width), -1)
    order, at = rng.permutation(blocks), 0
    for r, n in enumerate(held):
        table[r, :n], at = order[at:at + n], at + n
    keys, values, ks, vs = cache_of(rng, blocks, kv, block, dim, form, spread)
    # places that no token was written to: any code, NaN of the floating point format among them
    for r, n in enumerate(lengths):
        if n % block:
            keys[table[r, n // block], :, n % block:] = 0x7F
            values[table[r, n // block], :, :, n % block:] = 0xFF
    q = rng.standard_normal((heads, int(rows.sum()) + padding, dim)).astype(np.float32)
    return dict(q=q, keys=keys, values=values, key_scales=ks, value_scales=vs, table=table, lengths=lengths, starts=starts, rows=rows)


def attend_on_gpu(rt, c, block, form, window=0, max_rows=None, workspace=None, stream=None, fill=7.0):
    heads, tokens, dim = c["q"].shape
    d = {k: ints(rt, c[k]) for k in ("table", "lengths", "starts", "rows")}
    data = [rt.DeviceArray.of(c[k]) for k in ("keys", "values", "key_scales", "value_scales")]
    dq, out = rt.DeviceArray.of(c["q"]), rt.DeviceArray.of(np.full((tokens, heads, dim), fill, np.float32))
    batch = rt.KvBatch(requests=len(c["rows"]), tokens=tokens, max_rows=max_rows or max(1, int(c["rows"].max())), block=block,
                       blocks=len(c["keys"]), width=c["table"].shape[1], **{k: v.ptr for k, v in d.items()})
    cache = rt.Kv8(*(a.ptr for a in data), c["keys"].shape[1], dim, form)
    if workspace == "own":
        workspace = rt.DeviceArray((max(16, rt.attention_kv8_workspace(batch, cache, heads)),), np.uint8)
    rt.attention_kv8(batch, cache, dq, heads, out, window, workspace, stream)
    rt.synchronize()
    return out.numpy()


def check_attention(rt, c, block, form, window=0, workspace=None, max_rows=None):
    got = attend_on_gpu(rt, c, block, form, window, max_rows, workspace)
    want = np.full(got.shape, 7.0)
    A = ref.attention(**c, block=block, form=form, window=window, out=want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), np.argwhere(np.isnan(got) != np.isnan(want))[:5]
    fine = np.isfinite(want)
    largest = np.abs(ref.decode(c["values"][np.isfinite(c["value_scales"]).all(1)], form))
    largest = np.nanmax(largest) * np.nanmax(c["value_scales"])
    err = np.max(np.abs(got[fine] - want[fine]))
    assert err <= bound(A, c["lengths"].max(), largest), (err, bound(A, c["lengths"].max(), largest))
    return got


BATCHES = {"one key": [(1, 1)], "one": [(100, 1)], "long": [(5000, 1)], "ragged": [(1, 1), (777, 1), (64, 1), (65, 1), (16, 1), (300, 1), (2049, 1)],
           "few rows": [(50, 2), (400, 3), (4, 4), (129, 2)], "prompt": [(130, 130)], "prompts": [(70, 70), (1, 1), (33, 33), (200, 200)],
           "chunk": [(900, 150)], "mixed": [(300, 1), (500, 90), (40, 1), (80, 80), (1000, 5), (20, 1)], "long chunk": [(4500, 40)]}


@pytest.mark.parametrize("form", [ref.INT8, ref.E4M3])
@pytest.mark.parametrize("batch", BATCHES)
@pytest.mark.parametrize("heads,kv,dim,block,window", [(8, 1, 64, 16, 0), (14, 2, 64, 64, 0), (4, 1, 128, 32, 0), (3, 3, 80, 128, 0),
                                                       (6, 2, 32, 16, 70), (4, 2, 256, 64, 0), (2, 1, 16, 32, 5), (24, 1, 112, 16, 0)])
def test_attention(rt, form, batch, heads, kv, dim, block, window):
    if sum(l * r for l, r in BATCHES[batch]) * heads * dim > 2e8:
        heads = kv * max(1, heads // kv // 2)
    rng = np.random.default_rng(dim + block + len(batch))
    check_attention(rt, attention_case(rng, BATCHES[batch], heads, kv, dim, block, form, padding=3), block, form, window)


@pytest.mark.parametrize("requests", [1, 63, 200, 1100])
def test_attention_of_many_requests(rt, requests):
    rng = np.random.default_rng(requests)
    batch = [(int(rng.integers(1, 200)), 1) for _ in range(requests)]
    batch[requests // 2] = (3000, 1)
    check_attention(rt, attention_case(rng, batch, 4, 1, 64, 16, ref.INT8), 16, ref.INT8, workspace="own")


@pytest.mark.parametrize("requests,heads,kv", [([(900, 1)], 4, 2), ([(70, 3), (40, 1)], 4, 2), ([(300, 1), (64, 1), (2000, 1), (5, 1)], 20, 1),
                                               ([(1 + i % 90, 1 + i % 7) for i in range(600)], 6, 1)])
@pytest.mark.parametrize("padding", [0, 1000])
def test_attention_in_tiles_of_few_rows(rt, requests, heads, kv, padding):
    # the kernel of many rows with few of them: many padding rows, groups of more than 16, hundreds of requests
    requests = [(max(n, r), r) for n, r in requests]
    rng = np.random.default_rng(len(requests))
    check_attention(rt, attention_case(rng, requests, heads, kv, 64, 16, ref.INT8, padding=padding), 16, ref.INT8, workspace="own")


@pytest.mark.parametrize("form", [ref.INT8, ref.E4M3])
@pytest.mark.parametrize("window", [0, 90])
@pytest.mark.parametrize("heads,kv,dim,block", [(8, 2, 64, 16), (4, 1, 128, 64), (6, 2, 80, 32)])
def test_attention_decoding_beside_a_prompt(rt, form, window, heads, kv, dim, block):
    # both kernels in one call
    rng = np.random.default_rng(dim)
    batch = [(int(rng.integers(1, 700)), 1) for _ in range(30)] + [(170, 60), (2500, 1), (61, 3)]
    check_attention(rt, attention_case(rng, batch, heads, kv, dim, block, form, padding=5), block, form, window)


@pytest.mark.parametrize("batch", ["ragged", "mixed"])
def test_attention_of_huge_values(rt, batch):
    # value scales of 2^100, scores of ordinary size from tiny keys and large queries
    rng = np.random.default_rng(8)
    c = attention_case(rng, BATCHES[batch], 4, 2, 64, 16, ref.INT8)
    c["value_scales"] *= np.float32(2.0 ** 100)
    c["key_scales"] *= np.float32(2.0 ** -70)
    c["q"] *= np.float32(2.0 ** 70)
    check_attention(rt, c, 16, ref.INT8)


@pytest.mark.parametrize("form", [ref.INT8, ref.E4M3])
@pytest.mark.parametrize("batch", ["ragged", "mixed"])
def test_attention_scales_far_apart(rt, form, batch):
    # blocks whose scales differ by factors up to a million
    rng = np.random.default_rng(9)
    c = attention_case(rng, BATCHES[batch], 4, 2, 64, 16, form)
    c["value_scales"] = np.exp2(rng.integers(-20, 1, c["value_scales"].shape)).astype(np.float32)
    c["key_scales"] = np.exp2(rng.integers(-20, -4, c["key_scales"].shape)).astype(np.float32)
    check_attention(rt, c, 16, form)


@pytest.mark.parametrize("batch", ["ragged", "mixed", "chunk"])
@pytest.mark.parametrize("size", [1e-30, 1e-3, 30.0])
def test_attention_query_sizes(rt, batch, size):
    # flat, and sharp with scores up to hundreds
    rng = np.random.default_rng(10)
    c = attention_case(rng, BATCHES[batch], 4, 2, 64, 32, ref.INT8)
    c["q"] *= np.float32(size)
    check_attention(rt, c, 32, ref.INT8)


@pytest.mark.parametrize("form", [ref.INT8, ref.E4M3])
@pytest.mark.parametrize("window", [0, 100])
@pytest.mark.parametrize("batch", ["ragged", "mixed", "chunk", "long chunk"])
def test_attention_spoilt_blocks(rt, form, window, batch):
    # scales of NaN, of keys in one block and of values in another: the rows that see them, and no other
    rng = np.random.default_rng(11)
    c = attention_case(rng, BATCHES[batch], 4, 2, 64, 16, form, padding=2)
    r = int(np.argmax(c["lengths"]))
    n = c["lengths"][r]
    c["key_scales"][c["table"][r, (n - 20) // 16], 0] = np.nan
    c["value_scales"][c["table"][r, (n - 120) // 16], 1] = np.nan
    c["value_scales"][c["table"][r, 0], 0] = np.inf
    got = check_attention(rt, c, 16, form, window)
    assert np.isnan(got).any() and not np.isnan(got).all()


@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("batch", ["ragged", "mixed", "prompt"])
def test_attention_spoilt_queries(rt, what, batch):
    rng = np.random.default_rng(12)
    c = attention_case(rng, BATCHES[batch], 4, 2, 64, 16, ref.INT8)
    c["q"][1, 2 % c["q"].shape[1], 3] = what
    got = check_attention(rt, c, 16, ref.INT8)
    assert np.isnan(got).sum() == 64


@pytest.mark.parametrize("form", [ref.INT8, ref.E4M3])
@pytest.mark.parametrize("batch", ["ragged", "mixed"])
def test_attention_table_entries_that_are_no_blocks(rt, form, batch):
    rng = np.random.default_rng(13)
    c = attention_case(rng, BATCHES[batch], 4, 2, 64, 16, form)
    for r, entry, bad in ((1, 2, -1), (1, 3, len(c["keys"])), (3, 0, 2 ** 31 - 1)):
        c["table"][r, entry] = bad
    got = check_attention(rt, c, 16, form)
    assert np.isnan(got).any() and not np.isnan(got).all()


def test_attention_passes_over_requests_that_do_not_fit(rt):
    # no rows, more rows than keys, keys past the table, rows past the arrays or before them, more than max_rows
    rng = np.random.default_rng(14)
    c = attention_case(rng, [(30, 2), (40, 2), (50, 2), (60, 2), (70, 2), (80, 2), (90, 2)], 4, 2, 64, 16, ref.INT8, padding=4)
    plain = {k: c[k].copy() for k in ("rows", "lengths", "starts")}
    width = c["table"].shape[1]
    c["rows"][0], c["lengths"][1], c["lengths"][2] = 0, 1, width * 16 + 1
    c["starts"] = c["starts"].copy()
    c["starts"][3], c["starts"][4], c["rows"][5] = -1, 17, 3
    skipped = [0, 1, 2, 3, 4, 5]
    got = attend_on_gpu(rt, c, 16, ref.INT8, max_rows=2)
    for r in skipped:
        plain["rows"][r] = 0
    want = np.full(got.shape, 7.0)
    A = ref.attention(**{**c, **plain}, block=16, form=ref.INT8, window=0, out=want)
    largest = 127 * c["value_scales"].max()
    assert np.max(np.abs(got - want)) <= bound(A, 90, largest)
    assert (got[:12] == 7.0).all() and (got[14:] == 7.0).all()


@pytest.mark.parametrize("batch", ["long", "ragged", "mixed", "chunk", "long chunk"])
def test_attention_is_repeatable(rt, batch):
    # the same bits every time, with a workspace of the caller's or the stream's
    rng = np.random.default_rng(15)
    c = attention_case(rng, BATCHES[batch], 8, 2, 64, 32, ref.INT8)
    first = attend_on_gpu(rt, c, 32, ref.INT8)
    for workspace in (None, "own", "own"):
        assert np.array_equal(attend_on_gpu(rt, c, 32, ref.INT8, workspace=workspace), first)


def test_attention_far_offsets(rt):
    # codes past 4 GiB from the start of the pool
    heads, kv, dim, block = 4, 2, 128, 64
    blocks = (5 << 30) // (kv * dim * block)
    rng = np.random.default_rng(16)
    dk, dv = (rt.DeviceArray((blocks, kv, block, dim), np.uint8) for _ in range(2))
    ks, vs = (rt.DeviceArray.of(np.full((blocks, kv), 2.0 ** -5, np.float32)) for _ in range(2))
    pages = np.array([blocks - 1, blocks - 2, 3, blocks // 2 + 5])
    small = cache_of(rng, 4, kv, block, dim, ref.INT8)
    size = kv * dim * block
    for i, page in enumerate(pages):
        for d, a in ((dk, small[0]), (dv, small[1])):
            rt.check(rt.library().lh_copy_to_device(d.ptr + int(page) * size, np.ascontiguousarray(a[i]).ctypes.data, size))
    q = rng.standard_normal((heads, 1, dim)).astype(np.float32)
    d = {"table": ints(rt, pages[None]), "lengths": ints(rt, [250]), "starts": ints(rt, [0, 1]), "rows": ints(rt, [1])}
    dq, out = rt.DeviceArray.of(q), rt.DeviceArray((1, heads, dim), np.float32)
    batch = rt.KvBatch(requests=1, tokens=1, max_rows=1, block=block, blocks=blocks, width=4, **{k: v.ptr for k, v in d.items()})
    rt.attention_kv8(batch, rt.Kv8(dk.ptr, dv.ptr, ks.ptr, vs.ptr, kv, dim, ref.INT8), dq, heads, out)
    want, flat = np.zeros((1, heads, dim)), np.full((4, kv), 2.0 ** -5, np.float32)
    A = ref.attention(q, small[0], small[1], flat, flat, np.arange(4)[None], [250], [0, 1], [1], block, ref.INT8, 0, want)
    assert np.max(np.abs(out.numpy() - want)) <= bound(A, 250, 127 * 2.0 ** -5)
    # and an append there
    dq2, dqkv = rt.DeviceArray((heads, 1, dim), np.float32), rt.DeviceArray.of(rng.standard_normal((1, heads + 2 * kv, dim)).astype(np.float32))
    slot, pos = ints(rt, [int(pages[0]) * block + 58]), ints(rt, [0])
    batch.positions, batch.slots = pos.ptr, slot.ptr
    one = rt.DeviceArray.of(np.ones((1, dim // 2), np.float32))
    rt.rope_kv8(batch, rt.Kv8(dk.ptr, dv.ptr, ks.ptr, vs.ptr, kv, dim, ref.INT8), dqkv, heads, 0, one, one, dq2)
    rt.synchronize()
    wk, wks = small[0][:1].copy(), np.full((1, kv), 2.0 ** -5, np.float32)
    ref.append(wk, wks, dqkv.numpy()[:, heads:heads + kv], np.array([58]), block, ref.INT8, False)
    got = np.empty_like(wk)
    rt.check(rt.library().lh_copy_to_host(got.ctypes.data, dk.ptr + int(pages[0]) * size, size))
    assert np.array_equal(got, wk)


# ------------------------------------------------------- the three together ---
def serve(rt, steps, requests, tokens, heads, kv, dim, block, blocks, width, form, step_of, check_every=1):
    """A serving loop; step_of(pool, fresh, qkv) runs one step and returns its outputs.  Checked against the plain forms."""
    rng = np.random.default_rng(17)
    positions = width * block
    cos, sin = tables(rng, positions, dim // 2)
    state = dict(lengths=np.zeros(requests, int), table=np.full((requests, width), -1), stack=np.arange(blocks)[::-1].copy(), count=blocks)
    keys, values = np.zeros((blocks, kv, block, dim), np.uint8), np.zeros((blocks, kv, dim, block), np.uint8)
    ks, vs = np.zeros((blocks, kv), np.float32), np.zeros((blocks, kv), np.float32)
    for fresh in steps:
        qkv = rng.standard_normal((tokens, heads + 2 * kv, dim)).astype(np.float32)
        plan = ref.assign(state["lengths"], fresh, state["table"], state["stack"], state["count"], block, width, blocks, tokens, tokens)
        state.update(lengths=plan["lengths"], table=plan["table"], stack=plan["free_blocks"], count=int(plan["free_left"][0]))
        at = np.maximum(plan["positions"], 0)
        turned = ref.rotated(qkv[:, :heads + kv], cos[at][:, None], sin[at][:, None])
        ref.append(keys, ks, turned[:, heads:], plan["slots"], block, form, False)
        ref.append(values, vs, qkv[:, heads + kv:], plan["slots"], block, form, True)
        want = np.full((tokens, heads, dim), 7.0)
        A = ref.attention(turned[:, :heads].transpose(1, 0, 2), keys, values, ks, vs, plan["table"], plan["lengths"], plan["starts"],
                          plan["rows"], block, form, 0, want)
        got, plan_got = step_of(fresh, qkv, cos, sin)
        for name in ("lengths", "rows", "starts", "positions", "slots", "table"):
            assert np.array_equal(plan_got[name], plan[name]), name
        largest = np.nanmax(np.abs(ref.decode(values, form))) * vs.max()
        assert np.max(np.abs(got - want)) <= bound(A, plan["lengths"].max(), largest)
    return state


class Loop:
    """The device side of serve()."""

    def __init__(self, rt, requests, tokens, heads, kv, dim, block, blocks, width, form):
        self.rt, self.shape = rt, (heads, tokens, dim)
        self.pool = rt.BlockPool(requests, tokens, block, blocks, width)
        self.cache = rt.BlockCache(self.pool, kv, dim, form)
        self.qkv = rt.DeviceArray((tokens, heads + 2 * kv, dim), np.float32)
        self.q, self.out = rt.DeviceArray((heads, tokens, dim), np.float32).zero(), rt.DeviceArray((tokens, heads, dim), np.float32)
        self.cos = self.sin = None

    def load(self, fresh, qkv, cos, sin):
        rt = self.rt
        if self.cos is None:
            self.cos, self.sin = rt.DeviceArray.of(cos), rt.DeviceArray.of(sin)
        for d, a in ((self.pool.fresh, np.asarray(fresh, np.int32)), (self.qkv, qkv), (self.out, np.full(self.out.shape, 7.0, np.float32))):
            rt.check(rt.library().lh_copy_to_device(d.ptr, np.ascontiguousarray(a).ctypes.data, d.nbytes))

    def launch(self, stream=None, workspace=None):
        rt, batch, cache = self.rt, self.pool.batch, self.cache.desc
        heads, _, dim = self.shape
        rt.kv_assign(batch, stream)
        rt.rope_kv8(batch, cache, self.qkv, heads, dim, self.cos, self.sin, self.q, stream)
        rt.attention_kv8(batch, cache, self.q, heads, self.out, 0, workspace, stream)

    def results(self):
        self.rt.synchronize()
        return self.out.numpy(), {n: getattr(self.pool, n).numpy() for n in ("lengths", "rows", "starts", "positions", "slots", "table")}


STEPS = [[40, 1, 0, 17], [1, 30, 1, 1], [1, 1, 90, -1], [1, -1, 1, 20], [1, 64, 1, 1], [-1, 1, 1, 1], [33, 1, 1, 1], [1, 1, -1, 1], [1, 1, 100, 1]]


@pytest.mark.parametrize("form", ["int8", "e4m3"])
def test_serving_loop(rt, form):
    sizes = (4, 110, 8, 2, 64, 16, 20, 10)        # the pool of 20 blocks runs short and is reused
    loop = Loop(rt, *sizes, form)

    def step(fresh, qkv, cos, sin):
        loop.load(fresh, qkv, cos, sin)
        loop.launch()
        return loop.results()
    serve(rt, STEPS, *sizes, rt.KV8_FORMATS[form], step)


@pytest.mark.parametrize("own_workspace", [False, True])
def test_serving_loop_captured(rt, own_workspace):
    # one graph of a whole step, replayed: lengths, tables and free blocks advance on the device
    sizes = (4, 110, 8, 2, 64, 16, 40, 10)
    loop, stream, graphs = Loop(rt, *sizes, "int8"), rt.Stream(), []
    workspace = None
    if own_workspace:
        workspace = rt.DeviceArray((max(16, rt.attention_kv8_workspace(loop.pool.batch, loop.cache.desc, 8)),), np.uint8)

    def step(fresh, qkv, cos, sin):
        loop.load(fresh, qkv, cos, sin)
        rt.synchronize()
        if len(graphs) == 0:
            loop.launch(stream.handle, workspace)                 # eager once: the stream's scratch
            stream.synchronize()
            graphs.append(None)
            return loop.results()
        if graphs[0] is None:
            graphs[0] = rt.Graph(stream, lambda: loop.launch(stream.handle, workspace))
        scratch = rt.DeviceArray((1 << 16,), np.float32).zero()   # other work of the program between replays
        rt.synchronize()
        graphs[0].launch()
        stream.synchronize()
        scratch.free()
        return loop.results()
    serve(rt, STEPS, *sizes, ref.INT8, step)
    graphs[0].close()
    stream.close()


def test_first_call_in_a_capture_needs_a_workspace(rt):
    rng = np.random.default_rng(18)
    c = attention_case(rng, [(5000, 1)], 8, 2, 64, 64, ref.INT8)
    stream = rt.Stream()
    d = {k: ints(rt, c[k]) for k in ("table", "lengths", "starts", "rows")}
    data = [rt.DeviceArray.of(c[k]) for k in ("keys", "values", "key_scales", "value_scales")]
    dq, out = rt.DeviceArray.of(c["q"]), rt.DeviceArray((1, 8, 64), np.float32)
    batch = rt.KvBatch(requests=1, tokens=1, max_rows=1, block=64, blocks=len(c["keys"]), width=c["table"].shape[1], **{k: v.ptr for k, v in d.items()})
    cache = rt.Kv8(*(a.ptr for a in data), 2, 64, ref.INT8)
    need = rt.attention_kv8_workspace(batch, cache, 8)
    if need:
        with pytest.raises(rt.LeafError, match="outside stream capture"):
            rt.Graph(stream, lambda: rt.attention_kv8(batch, cache, dq, 8, out, stream=stream.handle))
        with pytest.raises(rt.LeafError, match="too small"):
            rt.check(rt.library().lh_attention_kv8(C.byref(batch), C.byref(cache), dq.ptr, 8, 0, out.ptr, out.ptr, need - 1, None))
    workspace = rt.DeviceArray((max(need, 16),), np.uint8)
    graph = rt.Graph(stream, lambda: rt.attention_kv8(batch, cache, dq, 8, out, 0, workspace, stream.handle))
    want = attend_on_gpu(rt, c, 64, ref.INT8)
    for _ in range(3):
        out.zero()
        rt.synchronize()
        graph.launch()
        stream.synchronize()
        assert np.array_equal(out.numpy(), want)
    graph.close()
    stream.close()


def test_two_streams_and_two_graphs(rt):
    # calls and graphs that may run at the same time: scratch of their streams, workspaces of their own
    rng = np.random.default_rng(19)
    cases = [attention_case(rng, b, 8, 2, 64, 32, ref.INT8) for b in ([(3000, 1)] * 6, [(2500, 1), (800, 1), (4000, 1)])]
    want = [attend_on_gpu(rt, c, 32, ref.INT8) for c in cases]
    streams, calls, outs, graphs, kept = [rt.Stream(), rt.Stream()], [], [], [], []
    for c in cases:
        heads, tokens, dim = c["q"].shape
        d = {k: ints(rt, c[k]) for k in ("table", "lengths", "starts", "rows")}
        data = [rt.DeviceArray.of(c[k]) for k in ("keys", "values", "key_scales", "value_scales")]
        batch = rt.KvBatch(requests=len(c["rows"]), tokens=tokens, max_rows=1, block=32, blocks=len(c["keys"]), width=c["table"].shape[1],
                           **{k: v.ptr for k, v in d.items()})
        cache = rt.Kv8(*(a.ptr for a in data), 2, dim, ref.INT8)
        q, out = rt.DeviceArray.of(c["q"]), rt.DeviceArray((tokens, heads, dim), np.float32)
        workspace = rt.DeviceArray((rt.attention_kv8_workspace(batch, cache, heads),), np.uint8)
        kept.append((d, data, q, workspace))
        outs.append(out)
        calls.append(lambda stream, workspace=None, a=(batch, cache, q, heads, out): rt.attention_kv8(*a, 0, workspace, stream))
    for _ in range(3):
        for out in outs:
            out.zero()
        rt.synchronize()
        for _ in range(4):
            for call, stream in zip(calls, streams):
                call(stream.handle)
        rt.synchronize()
        assert all(np.array_equal(o.numpy(), w) for o, w in zip(outs, want))
    for call, k in zip(calls, kept):
        graphs.append(rt.Graph(streams[0], lambda: call(streams[0].handle, k[3])))
    for _ in range(3):
        for out in outs:
            out.zero()
        rt.synchronize()
        for graph, stream in zip(graphs, streams):
            rt.check(rt.library().lh_graph_launch(graph.handle, stream.handle))
        rt.synchronize()
        assert all(np.array_equal(o.numpy(), w) for o, w in zip(outs, want))
    for g in graphs + streams:
        g.close()


@pytest.mark.parametrize("on_stream", [False, True])
def test_pool_steps_without_waits(rt, on_stream):
    # each step's new tokens are the ones given with it, on the default stream and on one of the library's
    requests, tokens, block, blocks, width = 5, 120, 16, 40, 9
    pool, stream = rt.BlockPool(requests, tokens, block, blocks, width), rt.Stream() if on_stream else None
    rng = np.random.default_rng(20)
    want = {"table": np.full((requests, width), -1), "free_blocks": np.arange(blocks)[::-1].copy(), "free_left": blocks,
            "lengths": np.zeros(requests, np.int64)}
    for i in range(20):
        fresh = rng.integers(0, 24, requests)
        if i % 3 == 2:
            fresh[i % requests] = -1
        pool.step(fresh, stream.handle if on_stream else None)
        want = ref.assign(want["lengths"], fresh, want["table"], want["free_blocks"], int(np.ravel(want["free_left"])[0]), block, width,
                          blocks, tokens, tokens)
    rt.synchronize()
    for name in ("lengths", "rows", "starts", "positions", "slots", "table"):
        assert np.array_equal(getattr(pool, name).numpy(), want[name]), name
    if on_stream:
        stream.close()

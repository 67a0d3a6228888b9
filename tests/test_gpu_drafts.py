"""Drafted trees over the 8-bit KV cache on the GPU against plain 64-bit forms (drafts_reference.py).

Plans, verification (its random numbers are hardly ever within rounding of a border, and the seeds are fixed),
scales, codes, lengths and blocks are equal.  Attention: the bound of test_gpu_kv8.py.
"""
from __future__ import annotations

import numpy as np
import pytest

from tests import drafts_reference as drafts
from tests import kv8_reference as ref
from tests import test_gpu_kv8 as kv8

pytestmark = pytest.mark.gpu
ints = kv8.ints


@pytest.fixture(scope="module")
def rt():
    from leaf_amd import runtime
    runtime.library()
    return runtime


# ------------------------------------------------------------------- plans ---
def tree_on_gpu(rt, parents, lengths, starts, rows, max_rows, block=16, width=1 << 16, stream=None):
    tokens, words = len(parents), -(-max_rows // 64)
    d = {k: ints(rt, a) for k, a in (("lengths", lengths), ("starts", starts), ("rows", rows), ("positions", np.full(tokens, -7)))}
    dp, masks = ints(rt, parents), rt.DeviceArray.of(np.full((tokens, words), 77, np.uint64))
    batch = rt.KvBatch(requests=len(rows), tokens=tokens, max_rows=max_rows, block=block, blocks=1, width=width, **{k: v.ptr for k, v in d.items()})
    rt.kv_tree(batch, dp, masks, stream)
    rt.synchronize()
    return d["positions"].numpy(), masks.numpy()


@pytest.mark.parametrize("counts,reach,extra", [([1], 1, 0), ([2, 1, 5], 3, 0), ([8] * 24, 2, 3), ([64, 63, 1], 9, 0), ([65, 130], 4, 0),
                                                ([512], 1, 0), ([511, 3, 200], 1000, 2), ([100] * 300, 5, 0), ([0, 7, 0, 1], 2, 1)])
def test_plans(rt, counts, reach, extra):
    rng = np.random.default_rng(len(counts) + reach)
    trees = [drafts.random_tree(rng, n, reach) if n else np.zeros(0, int) for n in counts]
    rows, cached = np.array(counts), rng.integers(0, 5000, len(counts))
    starts = np.concatenate([[0], np.cumsum(rows)])
    parents = np.concatenate(trees + [np.zeros(extra, int)])
    max_rows = min(512, max(counts) + extra)
    positions, masks = tree_on_gpu(rt, parents, cached + rows, starts, rows, max_rows)
    want, want_masks = np.full(len(parents), -7), np.full(masks.shape, 77, np.uint64)
    for r, tree in enumerate(trees):
        if len(tree):
            depth, seen = drafts.plan(tree)
            want[starts[r]:starts[r + 1]], want_masks[starts[r]:starts[r + 1]] = cached[r] + depth, drafts.packed(seen, masks.shape[1])
    assert np.array_equal(positions, want) and np.array_equal(masks, want_masks)


def test_plans_of_bad_arrays(rt):
    # parents that are no earlier rows stand for the cached text; requests that do not fit are passed over
    parents = np.array([0, 1, 5, -9, 2 ** 31 - 1, 1] * 4)
    positions, masks = tree_on_gpu(rt, parents, [50, 3, 2 ** 31 - 1, 90], [0, 6, 12, 19, 24], [6, 6, 6, 6], 6)
    depth, seen = drafts.plan(parents[:6])
    assert list(depth) == [0, 0, 0, 0, 0, 1]
    assert np.array_equal(positions[:6], 44 + depth) and np.array_equal(masks[:6], drafts.packed(seen, 1))
    assert (positions[6:] == -7).all() and (masks[6:] == 77).all()


# --------------------------------------------------------------- attention ---
def tree_case(rng, requests, heads, kv, dim, block, form, reach=3, padding=0, spread=0.5):
    """requests: (length, rows) each; a tree behind each request's cached keys."""
    c = kv8.attention_case(rng, requests, heads, kv, dim, block, form, padding, spread)
    c["seen"], c["positions"] = [], np.full(c["q"].shape[1], -1)
    for r, n in enumerate(c["rows"]):
        depth, seen = drafts.plan(drafts.random_tree(rng, n, reach))
        c["seen"].append(seen)
        c["positions"][c["starts"][r]:c["starts"][r] + n] = c["lengths"][r] - n + depth
    return c


def attend_on_gpu(rt, c, block, form, window=0, max_rows=None, workspace=None, stream=None, fill=7.0):
    heads, tokens, dim = c["q"].shape
    max_rows = max_rows or max(1, int(c["rows"].max()))
    words = -(-max_rows // 64)
    packed = np.full((tokens, words), 2 ** 64 - 1, np.uint64)
    for r, seen in enumerate(c["seen"]):
        if 0 <= c["starts"][r] <= tokens - len(seen):
            packed[c["starts"][r]:c["starts"][r] + len(seen)] = drafts.packed(seen, words)
    if c.get("garbage"):                            # bits of rows that a request does not have
        for r, seen in enumerate(c["seen"]):
            for j in range(len(seen), 64 * words):
                packed[c["starts"][r]:c["starts"][r] + len(seen), j // 64] |= np.uint64(1) << np.uint64(j % 64)
    d = {k: ints(rt, c[k]) for k in ("table", "lengths", "starts", "rows", "positions")}
    if not window:
        del d["positions"]
    data = [rt.DeviceArray.of(c[k]) for k in ("keys", "values", "key_scales", "value_scales")]
    dq, out, masks = rt.DeviceArray.of(c["q"]), rt.DeviceArray.of(np.full((tokens, heads, dim), fill, np.float32)), rt.DeviceArray.of(packed)
    batch = rt.KvBatch(requests=len(c["rows"]), tokens=tokens, max_rows=max_rows, block=block, blocks=len(c["keys"]),
                       width=c["table"].shape[1], **{k: v.ptr for k, v in d.items()})
    cache = rt.Kv8(*(a.ptr for a in data), c["keys"].shape[1], dim, form)
    if workspace == "own":
        workspace = rt.DeviceArray((max(16, rt.attention_kv8_tree_workspace(batch, cache, heads)),), np.uint8)
    rt.attention_kv8_tree(batch, cache, dq, heads, masks, out, window, workspace, stream)
    rt.synchronize()
    return out.numpy()


def check_attention(rt, c, block, form, window=0, workspace=None, max_rows=None):
    got = attend_on_gpu(rt, c, block, form, window, max_rows, workspace)
    want = np.full(got.shape, 7.0)
    A = drafts.attention(**{k: v for k, v in c.items() if k != "garbage"}, block=block, form=form, window=window, out=want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), np.argwhere(np.isnan(got) != np.isnan(want))[:5]
    fine = np.isfinite(want)
    largest = np.abs(ref.decode(c["values"][np.isfinite(c["value_scales"]).all(1)], form))
    largest = np.nanmax(largest) * np.nanmax(c["value_scales"])
    err = np.max(np.abs(got[fine] - want[fine]))
    assert err <= kv8.bound(A, c["lengths"].max(), largest), (err, kv8.bound(A, c["lengths"].max(), largest))
    return got


BATCHES = {"one": [(1, 1)], "single": [(300, 1), (64, 1), (2049, 1)], "small": [(50, 2), (400, 3), (4, 4), (129, 2), (7, 5)],
           "trees": [(64, 8), (900, 8), (71, 7), (8, 8), (1500, 5)], "wide": [(1100, 64), (64, 64), (700, 33), (100, 1)],
           "past a word": [(500, 130), (65, 65), (66, 1)], "large": [(700, 300)], "long": [(5000, 9)]}


@pytest.mark.parametrize("form", [ref.INT8, ref.E4M3])
@pytest.mark.parametrize("batch", BATCHES)
@pytest.mark.parametrize("heads,kv,dim,block,window", [(8, 1, 64, 16, 0), (14, 2, 64, 64, 0), (4, 1, 128, 32, 0), (3, 3, 80, 128, 0),
                                                       (6, 2, 32, 16, 70), (4, 2, 256, 64, 0), (2, 1, 16, 32, 3), (20, 1, 112, 16, 0)])
def test_attention(rt, form, batch, heads, kv, dim, block, window):
    if sum(l * r for l, r in BATCHES[batch]) * heads * dim > 2e8:
        heads = kv * max(1, heads // kv // 2)
    rng = np.random.default_rng(dim + block + len(batch))
    check_attention(rt, tree_case(rng, BATCHES[batch], heads, kv, dim, block, form, padding=3), block, form, window)


@pytest.mark.parametrize("requests,heads,kv", [([(900, 1)], 4, 2), ([(300, 1), (64, 1), (2000, 1), (5, 1)], 20, 1),
                                               ([(1 + i % 90, 1 + i % 7) for i in range(600)], 6, 1)])
@pytest.mark.parametrize("padding", [0, 1000])
def test_attention_of_other_routes(rt, requests, heads, kv, padding):
    # many padding rows, groups of more than 16, hundreds of requests
    rng = np.random.default_rng(len(requests))
    c = tree_case(rng, [(max(n, r), r) for n, r in requests], heads, kv, 64, 16, ref.INT8, padding=padding)
    check_attention(rt, c, 16, ref.INT8, workspace="own", max_rows=int(c["rows"].max()) + padding // 10)


@pytest.mark.parametrize("form", [ref.INT8, ref.E4M3])
@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("batch", ["small", "trees", "wide", "past a word", "long"])
def test_attention_of_any_masks(rt, form, window, batch):
    # masks that are no tree's: later rows, none at all, bits of rows that are not there; positions in any order
    rng = np.random.default_rng(21)
    c = tree_case(rng, BATCHES[batch] + [(6, 6)], 4, 2, 64, 16, form)
    c["seen"] = [rng.random(s.shape) < 0.4 for s in c["seen"]]
    for s in c["seen"]:
        s[-1] = False
    before = np.repeat(c["lengths"] - c["rows"], c["rows"])
    c["positions"] = before + rng.integers(-3, 60, len(before))
    c["garbage"] = True
    got = check_attention(rt, c, 16, form, window)
    # the last request has no cached key: a row without a bit sees none
    assert (got[-1] == 0).all()


@pytest.mark.parametrize("batch", ["trees", "wide"])
def test_attention_of_a_chain_is_causal(rt, batch):
    # a path of rows: what lh_attention_kv8 gives, to the rounding of both
    rng = np.random.default_rng(22)
    c = tree_case(rng, BATCHES[batch], 4, 2, 64, 16, ref.INT8, reach=1)
    got = check_attention(rt, c, 16, ref.INT8)
    plain = kv8.attend_on_gpu(rt, {k: v for k, v in c.items() if k not in ("seen", "positions")}, 16, ref.INT8)
    assert np.max(np.abs(got - plain)) < 1e-4


@pytest.mark.parametrize("form", [ref.INT8, ref.E4M3])
@pytest.mark.parametrize("window", [0, 30])
def test_attention_spoilt_blocks(rt, form, window):
    # scales of NaN in blocks of the step's own rows and of cached keys: the rows that see a key of them, and no other
    rng = np.random.default_rng(23)
    c = tree_case(rng, [(200, 40), (90, 20), (300, 64), (50, 3)], 4, 2, 64, 16, form, reach=30)
    c["key_scales"][c["table"][0, 195 // 16], 0] = np.nan
    c["value_scales"][c["table"][1, 80 // 16], 1] = np.inf
    c["value_scales"][c["table"][2, 10 // 16], 0] = -1.0
    c["table"][3, 1] = len(c["keys"])
    got = check_attention(rt, {**c, "value_scales": np.where(c["value_scales"] < 0, np.nan, c["value_scales"]).astype(np.float32)}, 16, form, window)
    raw = attend_on_gpu(rt, c, 16, form, window)
    assert np.array_equal(np.isnan(raw), np.isnan(got)) and np.isnan(got).any() and not np.isnan(got).all()


@pytest.mark.parametrize("what", [np.nan, np.inf])
def test_attention_spoilt_queries(rt, what):
    # a query that is not finite spoils its row, but one that sees no key
    rng = np.random.default_rng(24)
    c = tree_case(rng, [(80, 20), (5, 5)], 4, 2, 64, 16, ref.INT8)
    c["seen"][1][2] = False
    c["q"][1, 7, 3] = c["q"][2, 22, 5] = what
    got = check_attention(rt, c, 16, ref.INT8)
    assert np.isnan(got).sum() == 64 and (got[22] == 0).all()


def test_attention_passes_over_requests_that_do_not_fit(rt):
    rng = np.random.default_rng(25)
    c = tree_case(rng, [(30, 2), (40, 2), (50, 2), (60, 2), (70, 2), (80, 2), (90, 2)], 4, 2, 64, 16, ref.INT8, padding=4)
    plain = {k: c[k].copy() for k in ("rows", "lengths", "starts")}
    c["rows"][0], c["lengths"][1], c["lengths"][2] = 0, 1, c["table"].shape[1] * 16 + 1
    c["starts"] = c["starts"].copy()
    c["starts"][3], c["starts"][4], c["rows"][5] = -1, 17, 3
    got = attend_on_gpu(rt, c, 16, ref.INT8, max_rows=2)
    plain["rows"][:6] = 0
    want = np.full(got.shape, 7.0)
    A = drafts.attention(**{**c, **plain}, block=16, form=ref.INT8, window=0, out=want)
    assert np.max(np.abs(got - want)) <= kv8.bound(A, 90, 127 * c["value_scales"].max())
    assert (got[:12] == 7.0).all() and (got[14:] == 7.0).all()


@pytest.mark.parametrize("batch", ["trees", "wide", "long", "past a word"])
def test_attention_is_repeatable(rt, batch):
    rng = np.random.default_rng(26)
    c = tree_case(rng, BATCHES[batch], 8, 2, 64, 32, ref.INT8)
    first = attend_on_gpu(rt, c, 32, ref.INT8)
    for workspace in (None, "own", "own"):
        assert np.array_equal(attend_on_gpu(rt, c, 32, ref.INT8, workspace=workspace), first)


# ------------------------------------------------------------ verification ---
def draft_case(rng, counts, vocab, reach, with_draft, temperature, padding=0, sharp=3.0):
    """Trees whose tokens come from the draft's distributions, or are among its best."""
    rows = np.array(counts)
    starts, tokens = np.concatenate([[0], np.cumsum(rows)]), int(rows.sum()) + padding
    logits = (sharp * rng.standard_normal((tokens, vocab))).astype(np.float32)
    draft = (logits + 0.6 * rng.standard_normal((tokens, vocab))).astype(np.float32)
    temperatures = np.full(len(rows), temperature, np.float32) if np.isscalar(temperature) else np.asarray(temperature, np.float32)
    parents, ids = np.full(tokens, -1), rng.integers(0, vocab, tokens)
    for r, n in enumerate(rows):
        if not n:
            continue
        parents[starts[r]:starts[r] + n] = drafts.random_tree(rng, n, reach)
        for i in range(1, n):
            q = drafts.softmax(draft[starts[r] + parents[starts[r] + i]], temperatures[r] or 0.05)
            ids[starts[r] + i] = rng.choice(vocab, p=q) if q is not None else 0
    return dict(logits=logits, draft_logits=draft if with_draft else None, ids=ids, parents=parents, temperatures=temperatures,
                accept=rng.random(tokens).astype(np.float32), sample=rng.random(len(rows)).astype(np.float32), starts=starts, rows=rows)


def verify_on_gpu(rt, c, max_rows=None, workspace=None, stream=None):
    tokens, vocab = c["logits"].shape
    d = {k: None if c[k] is None else rt.DeviceArray.of(c[k]) for k in ("logits", "draft_logits", "temperatures", "accept", "sample")}
    d.update({k: ints(rt, c[k]) for k in ("ids", "parents")})
    d.update(path=ints(rt, np.full(tokens, -7)), kept=ints(rt, np.full(len(c["rows"]), -7)), next=ints(rt, np.full(len(c["rows"]), -7)))
    starts, rows = ints(rt, c["starts"]), ints(rt, c["rows"])
    batch = rt.KvBatch(requests=len(c["rows"]), tokens=tokens, max_rows=max_rows or max(1, int(max(c["rows"]))), block=16, blocks=1, width=1,
                       starts=starts.ptr, rows=rows.ptr)
    given = rt.Drafts(vocab=vocab, **{k: None if v is None else v.ptr for k, v in d.items()})
    if workspace == "own":
        workspace = rt.DeviceArray((max(16, rt.verify_drafts_workspace(batch, given)),), np.uint8)
    rt.verify_drafts(batch, given, workspace, stream)
    rt.synchronize()
    return d["path"].numpy(), d["kept"].numpy(), d["next"].numpy()


def check_verify(rt, c, workspace=None, max_rows=None):
    tokens = len(c["logits"])
    path, kept, following = np.full(tokens, -7), np.zeros(len(c["rows"]), int), np.full(len(c["rows"]), -1)
    for r, n in enumerate(c["rows"]):
        if n <= 0:
            continue
        own = slice(c["starts"][r], c["starts"][r] + n)
        one, following[r] = drafts.verify(c["logits"][own], None if c["draft_logits"] is None else c["draft_logits"][own], c["ids"][own],
                                          c["parents"][own], c["temperatures"][r], c["accept"][own], c["sample"][r])
        path[own] = -1
        path[own.start:own.start + len(one)], kept[r] = one, len(one)
    got = verify_on_gpu(rt, c, max_rows, workspace)
    for g, w, name in zip(got, (path, kept, following), ("path", "kept", "next")):
        assert np.array_equal(g, w), (name, np.argwhere(g != w)[:5], g[g != w][:5], w[g != w][:5])
    return kept, following


@pytest.mark.parametrize("with_draft", [False, True])
@pytest.mark.parametrize("vocab", [1, 2, 15, 17, 100, 1000, 1025, 32000, 50257])
@pytest.mark.parametrize("counts,reach", [([1], 1), ([5, 1, 3], 1), ([8] * 20, 3), ([26, 13, 0, 1], 5), ([70], 60)])
def test_verification(rt, counts, reach, vocab, with_draft):
    rng = np.random.default_rng(vocab + len(counts))
    temperature = np.where(np.arange(len(counts)) % 4 == 3, 0.0, rng.uniform(0.3, 1.5, len(counts)))
    kept, _ = check_verify(rt, draft_case(rng, counts, vocab, reach, with_draft, temperature, padding=2))
    if len(counts) == 20 and vocab == 32000:
        assert kept.max() > 2 and kept.min() < 3           # some stand, some do not


def test_verification_over_the_largest_vocabulary(rt):
    rng = np.random.default_rng(31)
    for with_draft in (False, True):
        check_verify(rt, draft_case(rng, [9, 4], 151936, 3, with_draft, [0.9, 1.1]))


@pytest.mark.parametrize("with_draft", [False, True])
@pytest.mark.parametrize("temperature,sharp", [(1e-3, 3.0), (1e-30, 3.0), (50.0, 3.0), (3e38, 1.0), (1.0, 0.0), (1.0, 200.0), (0.7, 1e30), (0.0, 0.0)])
def test_verification_temperatures(rt, temperature, sharp, with_draft):
    # one token has everything, all have the same, ties
    rng = np.random.default_rng(32)
    with np.errstate(over="ignore"):
        check_verify(rt, draft_case(rng, [6, 9, 1], 777, 2, with_draft, temperature, sharp=sharp))


@pytest.mark.parametrize("with_draft", [False, True])
def test_verification_random_numbers(rt, with_draft):
    # the least and the largest numbers of [0, 1); rows that stand without a test; what is outside
    rng = np.random.default_rng(33)
    for accept, sample in ((0.0, 0.0), (1 - 2.0 ** -24, 1 - 2.0 ** -24), (-1.0, 0.5), (1.0, 1.0), (np.nan, 2.0), (0.3, -1.0)):
        c = draft_case(rng, [7, 12, 1], 500, 2, with_draft, [0.8, 0.0, 1.0])
        c["accept"][:], c["sample"][:] = accept, sample
        kept, _ = check_verify(rt, c)
        if accept == -1.0:                                  # the first child of every row stands
            assert kept[0] >= 2
    c = draft_case(rng, [300], 500, 1, with_draft, 0.8)     # a prompt, all of whose rows stand, and a sampled token
    c["accept"][:] = -0.5
    assert check_verify(rt, c)[0][0] == 300


@pytest.mark.parametrize("with_draft", [False, True])
@pytest.mark.parametrize("greedy", [False, True])
def test_verification_masked_and_spoilt_logits(rt, with_draft, greedy):
    # minus infinity and the lowest value in most places; rows of NaN, of plus infinity and of nothing, which end a walk
    rng = np.random.default_rng(34)
    for what in (-np.inf, np.finfo(np.float32).min):
        c = draft_case(rng, [8] * 12, 300, 2, with_draft, 0.0 if greedy else 0.9)
        c["logits"][rng.random(c["logits"].shape) < 0.95] = what
        check_verify(rt, c)
        c["logits"][5] = c["logits"][30, 100:] = what
        c["logits"][30, :100] = what
        c["logits"][17, 299], c["logits"][26, 0], c["logits"][40:48, 7] = np.nan, np.inf, np.nan
        if with_draft:
            c["draft_logits"][65, 3], c["draft_logits"][72], c["draft_logits"][80:88, :290] = np.nan, -np.inf, -np.inf
        _, following = check_verify(rt, c)
        assert following[5] == -1                           # (its first row is NaN)


def test_verification_of_bad_tokens_and_temperatures(rt):
    rng = np.random.default_rng(35)
    for with_draft in (False, True):
        c = draft_case(rng, [8] * 6, 300, 2, with_draft, [0.9, -1.0, np.nan, np.inf, 0.0, 1.0])
        c["ids"][1::3], c["ids"][2::7] = 300, -1
        _, following = check_verify(rt, c)
        assert list(following[1:4]) == [-1, -1, -1]
    c = draft_case(rng, [20], 50, 30, False, 1.0)           # the same token for every child
    c["ids"][:], c["parents"][1:] = 3, 0
    check_verify(rt, c)


def test_verification_passes_over_requests_that_do_not_fit(rt):
    rng = np.random.default_rng(36)
    c = draft_case(rng, [4, 4, 4, 4, 4], 100, 2, True, 1.0, padding=3)
    c["rows"], c["starts"] = c["rows"].copy(), c["starts"].copy()
    c["rows"][0], c["rows"][1], c["starts"][2], c["starts"][3] = -3, 5, -1, 20
    path, kept, following = verify_on_gpu(rt, c, max_rows=4)
    assert list(kept[:4]) == [0] * 4 and list(following[:4]) == [-1] * 4 and kept[4] >= 1
    assert (path[:16] == -7).all() and (path[20:] == -7).all() and path[16] == 0


def test_verification_is_repeatable_and_shared(rt):
    # two streams at once, workspaces of the stream's and the caller's
    rng = np.random.default_rng(37)
    c = draft_case(rng, [9] * 30, 5000, 3, True, 0.8)
    first, streams = verify_on_gpu(rt, c), [rt.Stream(), rt.Stream()]
    for workspace, stream in ((None, streams[0]), ("own", streams[1]), ("own", streams[0])):
        assert all(np.array_equal(a, b) for a, b in zip(first, verify_on_gpu(rt, c, workspace=workspace, stream=stream.handle)))
    for s in streams:
        s.close()


# ----------------------------------------------------------------- keeping ---
def keep_case(rng, requests, kv, dim, block, form, layers, spread=2.0):
    """requests: (length, rows, kept path) each."""
    lengths, rows = np.array([q[0] for q in requests]), np.array([q[1] for q in requests])
    starts, kept = np.concatenate([[0], np.cumsum(rows)]), np.array([len(q[2]) for q in requests])
    path = np.full(int(rows.sum()) + 2, -1)
    for r, q in enumerate(requests):
        path[starts[r]:starts[r] + len(q[2])] = q[2]
    held = -(-lengths // block)
    blocks, width = int(held.sum()) + 2, int(held.max()) + 1
    table, order, at = np.full((len(rows), width), -1), rng.permutation(blocks), 0
    for r, n in enumerate(held):
        table[r, :n], at = order[at:at + n], at + n
    stack = np.full(blocks, -1)
    stack[:blocks - at] = order[at:]
    caches = [kv8.cache_of(rng, blocks, kv, block, dim, form, spread) for _ in range(layers)]
    return dict(lengths=lengths, rows=rows, starts=starts, kept=kept, path=path, table=table, stack=stack, count=blocks - at, caches=caches)


def random_paths(rng, requests):
    """Of (cached, rows): a kept path that ascends from row 0."""
    out = []
    for cached, n in requests:
        own = np.sort(rng.choice(np.arange(1, n), int(rng.integers(0, n)), replace=False)) if n > 1 else np.zeros(0, int)
        out.append((cached + n, n, [0, *own.tolist()]))
    return out


def check_keep(rt, c, block, form, in_place=True):
    kv, dim = c["caches"][0][0].shape[1], c["caches"][0][0].shape[3]
    blocks, tokens = len(c["stack"]), len(c["path"])
    d = {"lengths": ints(rt, c["lengths"]), "rows": ints(rt, c["rows"]), "starts": ints(rt, c["starts"]), "table": ints(rt, c["table"]),
         "free_blocks": ints(rt, c["stack"]), "free_count": ints(rt, [c["count"]]), "free_left": ints(rt, [-7])}
    after = d["lengths"] if in_place else ints(rt, np.full(len(c["rows"]), -7))
    if in_place:
        d["free_left"] = d["free_count"]
    path, kept = ints(rt, c["path"]), ints(rt, c["kept"])
    batch = rt.KvBatch(requests=len(c["rows"]), tokens=tokens, max_rows=max(1, min(512, int(c["rows"].max()))), block=block, blocks=blocks,
                       width=c["table"].shape[1], **{k: v.ptr for k, v in d.items()})
    data = [[rt.DeviceArray.of(a) for a in cache] for cache in c["caches"]]
    rt.kv8_compact(batch, [rt.Kv8(*(a.ptr for a in cache), kv, dim, form) for cache in data], path, kept)
    rt.kv_keep(batch, kept, None if in_place else after)
    rt.synchronize()
    for cache, got in zip(c["caches"], data):
        want = [a.copy() for a in cache]
        for i, transposed in ((0, False), (1, True)):
            drafts.compact(want[i], want[2 + i], c["table"], c["lengths"], c["starts"], c["rows"], c["path"], c["kept"], block, form, transposed)
        for g, w, name in zip(got, want, ("keys", "values", "key scales", "value scales")):
            g = g.numpy()
            assert np.array_equal(g, w, equal_nan=g.dtype == np.float32), (name, np.argwhere(g != w)[:4])
    lengths, stack, count = drafts.keep(c["lengths"], c["rows"], c["kept"], c["table"], c["stack"], c["count"], block, blocks)
    assert np.array_equal(after.numpy(), lengths) and d["free_left"].numpy()[0] == count
    assert np.array_equal(d["free_blocks"].numpy(), stack)


@pytest.mark.parametrize("form", [ref.INT8, ref.E4M3])
@pytest.mark.parametrize("kv,dim,block,layers", [(2, 64, 16, 3), (1, 128, 64, 2), (3, 80, 32, 1), (5, 16, 128, 35), (2, 256, 128, 1)])
def test_keeping(rt, form, kv, dim, block, layers):
    rng = np.random.default_rng(dim + block)
    requests = [(0, 1), (5, 8), (15, 8), (16, 3), (40, 26), (3, 64), (127, 70), (0, 200), (9, 2)]
    check_keep(rt, keep_case(rng, random_paths(rng, requests), kv, dim, block, form, layers), block, form, in_place=layers != 2)


@pytest.mark.parametrize("form", [ref.INT8, ref.E4M3])
def test_keeping_in_place_and_nothing(rt, form):
    # paths that move nothing leave every code and scale; kept 0 gives all of a step's blocks back
    rng = np.random.default_rng(41)
    c = keep_case(rng, [(40, 9, [0, 1, 2]), (33, 33, list(range(33))), (50, 20, [0]), (64, 64, [0, 63])], 2, 64, 16, form, 2)
    check_keep(rt, c, 16, form)
    c["kept"][:] = 0
    check_keep(rt, c, 16, form)


def test_keeping_bad_paths(rt):
    # paths that do not ascend, leave the rows or are longer than them; kept out of range; blocks that are none
    rng = np.random.default_rng(42)
    c = keep_case(rng, [(40, 9, [0, 4, 2]), (33, 9, [0, 3, 3]), (50, 9, [0, 9]), (64, 9, [-1, 2]), (70, 9, [0, 5]), (80, 9, [1, 5, 8]), (90, 9, [0, 2, 4]),
                        (45, 20, [0, 5, 17])], 2, 64, 16, ref.INT8, 2)
    c["kept"][4] = 10
    c["kept"][6] = -1
    c["table"][5, 4] = -1                                   # rows 71..79 begin in block 4
    c["table"][7, 2] = 10 ** 6                              # its last rows' block
    check_keep(rt, c, 16, ref.INT8)


@pytest.mark.parametrize("form", [ref.INT8, ref.E4M3])
def test_keeping_spoilt_scales(rt, form):
    rng = np.random.default_rng(43)
    c = keep_case(rng, [(40, 20, [0, 3, 9, 19]), (31, 16, [0, 15]), (70, 30, [0, 1, 2, 29])], 2, 64, 16, form, 1)
    keys, values, ks, vs = c["caches"][0]
    ks[c["table"][0, 2], 0], vs[c["table"][1, 0], 1], ks[c["table"][2, 4], 1] = np.nan, -2.0, np.inf
    check_keep(rt, c, 16, form)


def test_keeping_bad_counts(rt):
    # a free count out of range, more blocks than the pool holds, lengths past the table: nothing is written out of bounds
    rng = np.random.default_rng(44)
    c = keep_case(rng, [(100, 90, [0]), (100, 90, [0]), (30, 5, [0]), (20, 3, [0])], 1, 16, 16, ref.INT8, 1)
    c["lengths"][2], c["rows"][3] = 10 ** 6, 30
    for count in (-5, len(c["stack"]) - 1, 2 ** 31 - 1):
        d = {k: ints(rt, c[k]) for k in ("lengths", "rows", "table")}
        stack, free, left, after = ints(rt, c["stack"]), ints(rt, [count]), ints(rt, [-7]), ints(rt, [-7] * 4)
        batch = rt.KvBatch(requests=4, tokens=200, max_rows=90, block=16, blocks=len(c["stack"]), width=c["table"].shape[1], free_blocks=stack.ptr,
                           free_count=free.ptr, free_left=left.ptr, **{k: v.ptr for k, v in d.items()})
        rt.kv_keep(batch, ints(rt, [1, 1, 1, 1]), after)
        rt.synchronize()
        assert left.numpy()[0] == min(len(c["stack"]), max(count, 0) + 12) and list(after.numpy()) == [11, 11, 10 ** 6, 20]


def test_keeping_many_requests(rt):
    rng = np.random.default_rng(45)
    requests = [(int(rng.integers(0, 100)), int(rng.integers(1, 40))) for _ in range(4000)]
    check_keep(rt, keep_case(rng, random_paths(rng, requests), 1, 16, 16, ref.INT8, 1), 16, ref.INT8)


@pytest.mark.parametrize("with_draft", [False, True])
@pytest.mark.parametrize("vocab", [5000, 32000, 50257])
def test_verification_without_waiting(rt, monkeypatch, vocab, with_draft):
    # a workgroup that waits for no other computes all that they owe it, to the same results
    monkeypatch.setenv("LEAF_VERIFY_WAIT", "0")
    rng = np.random.default_rng(vocab)
    for counts in ([6], [8] * 40):
        check_verify(rt, draft_case(rng, counts, vocab, 3, with_draft, np.where(np.arange(len(counts)) % 5 == 4, 0.0, 0.9), padding=1))

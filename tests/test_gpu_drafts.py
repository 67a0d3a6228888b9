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


@pytest.mark.parametrize("form", [ref.INT8, ref.E4M3])
@pytest.mark.parametrize("heads,kv,dim,block", [(6, 2, 192, 32), (8, 2, 176, 64), (4, 1, 240, 16), (6, 2, 144, 128), (6, 3, 48, 16), (80, 1, 64, 64)])
def test_attention_of_other_heads(rt, form, heads, kv, dim, block):
    # up to 32 rows of a KV head, and more
    rng = np.random.default_rng(dim + heads)
    for batch in ([(700, 6), (90, 7), (6, 6)], [(500, 33), (150, 20), (1100, 7)]):
        check_attention(rt, tree_case(rng, batch, heads, kv, dim, block, form, padding=1), block, form)


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


@pytest.mark.parametrize("form", [ref.INT8, ref.E4M3])
@pytest.mark.parametrize("batch", ["small", "trees", "wide", "long"])
def test_attention_scales_far_apart(rt, form, batch):
    # blocks whose scales differ by factors up to a million; then huge values under scores of ordinary size
    rng = np.random.default_rng(27)
    c = tree_case(rng, BATCHES[batch], 4, 2, 64, 16, form)
    c["value_scales"] = np.exp2(rng.integers(-20, 1, c["value_scales"].shape)).astype(np.float32)
    c["key_scales"] = np.exp2(rng.integers(-20, -4, c["key_scales"].shape)).astype(np.float32)
    check_attention(rt, c, 16, form)
    c = tree_case(rng, BATCHES[batch], 4, 2, 64, 16, form)
    c["value_scales"] *= np.float32(2.0 ** 100)
    c["key_scales"] *= np.float32(2.0 ** -70)
    c["q"] *= np.float32(2.0 ** 70)
    check_attention(rt, c, 16, form)


@pytest.mark.parametrize("batch", ["small", "trees", "wide"])
@pytest.mark.parametrize("size", [1e-30, 1e-3, 30.0])
def test_attention_query_sizes(rt, batch, size):
    # flat, and sharp with scores up to hundreds
    rng = np.random.default_rng(28)
    c = tree_case(rng, BATCHES[batch], 4, 2, 64, 32, ref.INT8)
    c["q"] *= np.float32(size)
    check_attention(rt, c, 32, ref.INT8)


@pytest.mark.parametrize("heads", [2, 16, 40])
def test_attention_of_scores_far_from_zero(rt, heads):
    # scores of 2^24 and more: of keys that are the same, whatever row of the step or cached key they are, each weighs alike
    rng = np.random.default_rng(29)
    for scale in (2.0 ** 10, -2.0 ** 12):
        c = tree_case(rng, [(90, 9), (40, 20)], heads, 1, 64, 16, ref.INT8)
        c["keys"][:] = c["keys"][0, 0, 0]
        c["key_scales"][:] = np.float32(2.0 ** 8)
        c["q"][:] = np.float32(scale) * ref.decode(c["keys"][0, 0, 0], ref.INT8).astype(np.float32)
        got = attend_on_gpu(rt, c, 16, ref.INT8)
        # equal scores: the mean of the values that a row sees; 90 weights of 2^-22, sums in f32, a value scale of 2^-3 at most
        values = ref.decode(c["values"], ref.INT8) * c["value_scales"][:, :, None, None]
        for r in range(2):
            v = values[c["table"][r, :-(-c["lengths"][r] // 16)], 0].transpose(0, 2, 1).reshape(-1, 64)[:c["lengths"][r]]
            before = c["lengths"][r] - c["rows"][r]
            for i in range(c["rows"][r]):
                want = v[np.concatenate([np.ones(before, bool), c["seen"][r][i]])].mean(0)
                assert np.abs(got[c["starts"][r] + i] - want).max() <= 2.0 ** -19 * np.abs(v).max()


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


# ------------------------------------------------------- all of them together ---
class Loop:
    """The device side of a serving loop with drafts: `layers` caches over one pool, a vocabulary, trees of up to `most` rows."""

    def __init__(self, rt, requests, tokens, most, heads, kv, dim, block, blocks, width, layers, vocab, form):
        self.rt, self.shape, self.vocab = rt, (heads, tokens, dim), vocab
        self.pool = rt.BlockPool(requests, tokens, block, blocks, width, max_rows=most)
        self.caches = [rt.BlockCache(self.pool, kv, dim, form) for _ in range(layers)]
        for cache in self.caches:                           # (codes and scales that no token wrote)
            for a in (cache.keys, cache.values, cache.key_scales, cache.value_scales):
                a.zero()
        floats = {"qkv": (layers, tokens, heads + 2 * kv, dim), "logits": (tokens, vocab), "draft_logits": (tokens, vocab),
                  "temperatures": (requests,), "accept": (tokens,), "sample": (requests,)}
        self.data = {k: rt.DeviceArray(s, np.float32) for k, s in floats.items()}
        self.data.update({k: rt.DeviceArray.of(np.full(n, -1, np.int32)) for k, n in
                          (("parents", tokens), ("ids", tokens), ("path", tokens), ("kept", requests), ("next", requests))})
        self.masks = rt.DeviceArray.of(np.zeros((tokens, -(-most // 64)), np.uint64))
        self.q = [rt.DeviceArray((heads, tokens, dim), np.float32).zero() for _ in range(layers)]
        self.out = [rt.DeviceArray((tokens, heads, dim), np.float32) for _ in range(layers)]
        self.drafts = rt.Drafts(vocab=vocab, **{k: self.data[k].ptr for k, _ in rt.Drafts._fields_[1:]})
        self.cos = self.sin = None
        rt.synchronize()

    def load(self, fresh, cos, sin, **data):
        rt = self.rt
        if self.cos is None:
            self.cos, self.sin = rt.DeviceArray.of(cos), rt.DeviceArray.of(sin)
        pairs = [(self.pool.fresh, np.asarray(fresh, np.int32))] + [(o, np.full(o.shape, 7.0, np.float32)) for o in self.out]
        for d, a in pairs + [(self.data[k], np.asarray(a, self.data[k].dtype)) for k, a in data.items()]:
            assert a.nbytes == d.nbytes
            rt.check(rt.library().lh_copy_to_device(d.ptr, np.ascontiguousarray(a).ctypes.data, d.nbytes))

    def launch(self, stream=None, workspaces=(None, None)):
        rt, batch, d = self.rt, self.pool.batch, self.data
        heads, _, dim = self.shape
        layer = d["qkv"].nbytes // len(self.caches)
        rt.kv_assign(batch, stream)
        rt.kv_tree(batch, d["parents"], self.masks, stream)
        for i, cache in enumerate(self.caches):
            rt.check(rt.library().lh_rope_kv8(batch, cache.desc, d["qkv"].ptr + i * layer, heads, dim, self.cos.ptr, self.sin.ptr,
                                              self.cos.shape[0], self.q[i].ptr, stream))
            rt.attention_kv8_tree(batch, cache.desc, self.q[i], heads, self.masks, self.out[i], 0, workspaces[0], stream)
        rt.verify_drafts(batch, self.drafts, workspaces[1], stream)
        rt.kv8_compact(batch, [c.desc for c in self.caches], d["path"], d["kept"], stream)
        rt.kv_keep(batch, d["kept"], stream=stream)

    def results(self):
        self.rt.synchronize()
        got = {n: getattr(self.pool, n).numpy() for n in ("lengths", "rows", "starts", "positions", "slots", "table", "free_blocks", "free_count")}
        got.update({n: self.data[n].numpy() for n in ("path", "kept", "next")})
        got["out"] = [o.numpy() for o in self.out]
        got["caches"] = [[a.numpy() for a in (c.keys, c.values, c.key_scales, c.value_scales)] for c in self.caches]
        return got


def serve(rt, loop, steps, requests, tokens, most, heads, kv, dim, block, blocks, width, layers, vocab, form, run):
    """Steps of trees (each request's rows; negative: it has ended), checked against the plain forms after every step."""
    rng = np.random.default_rng(51)
    cos, sin = kv8.tables(rng, width * block, dim // 2)
    lengths, table, stack, count = np.zeros(requests, int), np.full((requests, width), -1), np.arange(blocks)[::-1].copy(), blocks
    caches = [[np.zeros(s, np.uint8) for s in ((blocks, kv, block, dim), (blocks, kv, dim, block))] +
              [np.zeros((blocks, kv), np.float32) for _ in range(2)] for _ in range(layers)]
    moved = 0
    for fresh in steps:
        c = draft_case(rng, [max(n, 0) for n in fresh], vocab, 3, True, rng.choice([0.0, 0.7, 1.2], requests),
                       padding=tokens - sum(max(n, 0) for n in fresh))
        qkv = rng.standard_normal((layers, tokens, heads + 2 * kv, dim)).astype(np.float32)
        given = {k: c[k] for k in ("logits", "draft_logits", "temperatures", "accept", "sample", "parents", "ids")}
        got = run(fresh, cos, sin, qkv=qkv, **given)
        plan = ref.assign(lengths, fresh, table, stack, count, block, width, blocks, tokens, most)
        starts, rows, table = plan["starts"], plan["rows"], plan["table"]
        seen, positions = [], plan["positions"].copy()
        for r in range(requests):
            own = slice(starts[r], starts[r] + rows[r])
            depth, ancestors = drafts.plan(c["parents"][own])
            seen.append(ancestors)
            positions[own] = plan["lengths"][r] - rows[r] + depth
        path, kept, following = got["path"].copy(), np.zeros(requests, int), np.full(requests, -1)
        for r in range(requests):
            if rows[r] == 0:
                continue
            own = slice(starts[r], starts[r] + rows[r])
            one, following[r] = drafts.verify(c["logits"][own], c["draft_logits"][own], c["ids"][own], c["parents"][own], c["temperatures"][r],
                                              c["accept"][own], c["sample"][r])
            path[own] = -1
            path[own.start:own.start + len(one)], kept[r] = one, len(one)
            moved += any(a != b for a, b in enumerate(one))
        at = np.maximum(positions, 0)
        for i in range(layers):
            keys, values, ks, vs = caches[i]
            turned = ref.rotated(qkv[i][:, :heads + kv], cos[at][:, None], sin[at][:, None])
            ref.append(keys, ks, turned[:, heads:], plan["slots"], block, form, False)
            ref.append(values, vs, qkv[i][:, heads + kv:], plan["slots"], block, form, True)
            want = np.full((tokens, heads, dim), 7.0)
            A = drafts.attention(turned[:, :heads].transpose(1, 0, 2), keys, values, ks, vs, table, plan["lengths"], starts, rows, seen, positions,
                                 block, form, 0, want)
            largest = np.nanmax(np.abs(ref.decode(values, form))) * vs.max()
            assert np.max(np.abs(got["out"][i] - want)) <= kv8.bound(A, plan["lengths"].max(), largest)
            for codes, scales, transposed in ((keys, ks, False), (values, vs, True)):
                drafts.compact(codes, scales, table, plan["lengths"], starts, rows, path, kept, block, form, transposed)
            for g, w in zip(got["caches"][i], caches[i]):
                assert np.array_equal(g, w)
        lengths, stack, count = drafts.keep(plan["lengths"], rows, kept, table, plan["free_blocks"], int(plan["free_left"][0]), block, blocks)
        for name, want in (("rows", rows), ("starts", starts), ("positions", positions), ("slots", plan["slots"]), ("table", table),
                           ("path", path), ("kept", kept), ("next", following), ("lengths", lengths), ("free_count", [count])):
            assert np.array_equal(got[name], want), name
        assert np.array_equal(got["free_blocks"][:count], stack[:count])
    assert moved > 3                                        # (some paths leave rows out)


SIZES = dict(requests=4, tokens=90, most=24, heads=8, kv=2, dim=64, block=16, blocks=24, width=8, layers=2, vocab=3000)
STEPS = [[20, 1, 0, 17], [8, 24, 8, 1], [8, 8, 23, -1], [7, -1, 5, 20], [8, 24, 1, 8], [-1, 8, 8, 8], [24, 8, 24, 24], [9, 9, -1, 9], [8, 1, 24, 8]]


@pytest.mark.parametrize("form", ["int8", "e4m3"])
def test_serving_loop(rt, form):
    loop = Loop(rt, *SIZES.values(), form)

    def run(fresh, cos, sin, **data):
        loop.load(fresh, cos, sin, **data)
        loop.launch()
        return loop.results()
    serve(rt, loop, STEPS, *SIZES.values(), rt.KV8_FORMATS[form], run)


@pytest.mark.parametrize("own_workspaces", [False, True])
def test_serving_loop_captured(rt, own_workspaces):
    # one graph of a whole step, replayed, with the program's own work and waits between
    loop, stream, graphs = Loop(rt, *SIZES.values(), "int8"), rt.Stream(), []
    spaces = (None, None)
    if own_workspaces:
        spaces = tuple(rt.DeviceArray((max(16, n),), np.uint8) for n in (
            rt.attention_kv8_tree_workspace(loop.pool.batch, loop.caches[0].desc, 8), rt.verify_drafts_workspace(loop.pool.batch, loop.drafts)))

    def run(fresh, cos, sin, **data):
        loop.load(fresh, cos, sin, **data)
        rt.synchronize()
        if not graphs and not own_workspaces:
            loop.launch(stream.handle, spaces)              # eager once: the stream's scratch
            stream.synchronize()
            graphs.append(None)
            return loop.results()
        if not graphs or graphs[0] is None:
            graphs[:] = [rt.Graph(stream, lambda: loop.launch(stream.handle, spaces))]
        between = rt.DeviceArray((1 << 16,), np.float32).zero()
        rt.synchronize()
        graphs[0].launch()
        stream.synchronize()
        between.free()
        return loop.results()
    serve(rt, loop, STEPS, *SIZES.values(), ref.INT8, run)
    graphs[0].close()
    stream.close()


def test_first_calls_in_a_capture_need_workspaces(rt):
    rng = np.random.default_rng(52)
    stream = rt.Stream()
    starts, rows = ints(rt, [0, 3]), ints(rt, [3])
    c = draft_case(rng, [3], 40000, 1, True, 0.9)
    d = {k: rt.DeviceArray.of(c[k]) for k in ("logits", "draft_logits", "temperatures", "accept", "sample")}
    d.update({k: ints(rt, c[k]) for k in ("ids", "parents")})
    d.update(path=ints(rt, [-7] * 3), kept=ints(rt, [-7]), next=ints(rt, [-7]))
    batch = rt.KvBatch(requests=1, tokens=3, max_rows=3, block=16, blocks=1, width=1, starts=starts.ptr, rows=rows.ptr)
    given = rt.Drafts(vocab=40000, **{k: v.ptr for k, v in d.items()})
    need = rt.verify_drafts_workspace(batch, given)
    assert need > 0
    with pytest.raises(rt.LeafError, match="outside stream capture"):
        rt.Graph(stream, lambda: rt.verify_drafts(batch, given, None, stream.handle))
    workspace = rt.DeviceArray((need,), np.uint8)
    with pytest.raises(rt.LeafError, match="too small"):
        rt.check(rt.library().lh_verify_drafts(batch, given, workspace.ptr, need - 1, None))
    want = drafts.verify(c["logits"], c["draft_logits"], c["ids"], c["parents"], c["temperatures"][0], c["accept"], c["sample"][0])
    graph = rt.Graph(stream, lambda: rt.verify_drafts(batch, given, workspace, stream.handle))
    for _ in range(3):
        rt.check(rt.library().lh_copy_to_device(d["next"].ptr, np.array([-7], np.int32).ctypes.data, 4))
        rt.synchronize()
        graph.launch()
        stream.synchronize()
        assert d["next"].numpy()[0] == want[1] and list(d["path"].numpy()[:len(want[0])]) == want[0]
    graph.close()
    stream.close()


def test_two_streams_at_once(rt):
    # attention and verification on two streams, in scratch of their streams and in workspaces of their own; then in two graphs
    rng = np.random.default_rng(53)
    streams, calls, outs, want, kept, graphs = [rt.Stream(), rt.Stream()], [], [], [], [], []
    for n, counts in enumerate(([9] * 12, [30, 5, 17])):
        c = tree_case(rng, [(1500 + 300 * i, r) for i, r in enumerate(counts)], 8, 2, 64, 32, ref.INT8)
        v = draft_case(rng, counts, 20000, 3, True, 0.8)
        want.append([attend_on_gpu(rt, c, 32, ref.INT8), *verify_on_gpu(rt, v)])
        tokens, words = len(v["ids"]), -(-max(counts) // 64)
        d = {k: ints(rt, c[k]) for k in ("table", "lengths", "starts", "rows")}
        data = [rt.DeviceArray.of(c[k]) for k in ("keys", "values", "key_scales", "value_scales", "q")]
        masks = rt.DeviceArray.of(np.concatenate([drafts.packed(s, words) for s in c["seen"]]))
        f = {k: rt.DeviceArray.of(v[k]) for k in ("logits", "draft_logits", "temperatures", "accept", "sample")}
        f.update({k: ints(rt, v[k]) for k in ("ids", "parents")})
        f.update(path=ints(rt, [0] * tokens), kept=ints(rt, [0] * len(counts)), next=ints(rt, [0] * len(counts)))
        out = rt.DeviceArray((tokens, 8, 64), np.float32)
        batch = rt.KvBatch(requests=len(counts), tokens=tokens, max_rows=max(counts), block=32, blocks=len(c["keys"]), width=c["table"].shape[1],
                           **{k: a.ptr for k, a in d.items()})
        cache = rt.Kv8(*(a.ptr for a in data[:4]), 2, 64, ref.INT8)
        given = rt.Drafts(vocab=20000, **{k: a.ptr for k, a in f.items()})
        spaces = [rt.DeviceArray((max(16, size),), np.uint8) for size in (rt.attention_kv8_tree_workspace(batch, cache, 8),
                                                                        rt.verify_drafts_workspace(batch, given))]
        kept.append((d, data, masks, f, spaces))
        outs.append((out, f["path"], f["kept"], f["next"]))

        def call(stream, own, a=(batch, cache, data[4], masks, out, given, spaces)):
            batch, cache, q, masks, out, given, spaces = a
            rt.attention_kv8_tree(batch, cache, q, 8, masks, out, 0, spaces[0] if own else None, stream)
            rt.verify_drafts(batch, given, spaces[1] if own else None, stream)
        calls.append(call)

    def check():
        rt.synchronize()
        for own, expected in zip(outs, want):
            assert all(np.array_equal(o.numpy(), w) for o, w in zip(own, expected))
            for o in own:
                o.zero()
        rt.synchronize()
    for own in (False, True):
        for _ in range(3):
            for call, stream in zip(calls, streams):
                call(stream.handle, own)
        check()
    for call in calls:
        graphs.append(rt.Graph(streams[0], lambda: call(streams[0].handle, True)))
    for _ in range(3):
        for graph, stream in zip(graphs, streams):
            rt.check(rt.library().lh_graph_launch(graph.handle, stream.handle))
        check()
    for g in graphs + streams:
        g.close()


# ------------------------------------------------------------- far offsets ---
def test_verification_far_offsets(rt):
    # logits past 2^31 values from the first
    vocab, tokens, first = 151936, 14500, 14200
    rng = np.random.default_rng(54)
    c = draft_case(rng, [7], vocab, 2, True, 0.9)
    logits, draft = (rt.DeviceArray((tokens, vocab), np.float32).zero() for _ in range(2))
    size = 4 * vocab
    for d, a in ((logits, c["logits"]), (draft, c["draft_logits"])):
        rt.check(rt.library().lh_copy_to_device(d.ptr + first * size, np.ascontiguousarray(a).ctypes.data, a.nbytes))
    ids, parents, accept = np.zeros(tokens, np.int32), np.full(tokens, -1, np.int32), np.zeros(tokens, np.float32)
    ids[first:first + 7], parents[first:first + 7], accept[first:first + 7] = c["ids"], c["parents"], c["accept"]
    d = {"ids": ints(rt, ids), "parents": ints(rt, parents), "accept": rt.DeviceArray.of(accept), "temperatures": rt.DeviceArray.of(c["temperatures"]),
         "sample": rt.DeviceArray.of(c["sample"]), "path": ints(rt, ids), "kept": ints(rt, [0]), "next": ints(rt, [0])}
    starts, rows = ints(rt, [first, tokens]), ints(rt, [7])
    batch = rt.KvBatch(requests=1, tokens=tokens, max_rows=7, block=16, blocks=1, width=1, starts=starts.ptr, rows=rows.ptr)
    rt.verify_drafts(batch, rt.Drafts(vocab=vocab, logits=logits.ptr, draft_logits=draft.ptr, **{k: v.ptr for k, v in d.items()}))
    rt.synchronize()
    path, following = drafts.verify(c["logits"], c["draft_logits"], c["ids"], c["parents"], c["temperatures"][0], c["accept"], c["sample"][0])
    assert d["kept"].numpy()[0] == len(path) and d["next"].numpy()[0] == following
    assert list(d["path"].numpy()[first:first + len(path)]) == path


def test_cache_far_offsets(rt):
    # codes past 4 GiB from the start of the pool: attention of a tree, then its rows kept
    heads, kv, dim, block = 4, 2, 128, 64
    blocks = (5 << 30) // (kv * dim * block)
    rng = np.random.default_rng(55)
    dk, dv = (rt.DeviceArray((blocks, kv, block, dim), np.uint8) for _ in range(2))
    flat = np.full((blocks, kv), 2.0 ** -5, np.float32)
    pages = np.array([blocks - 1, 3, blocks - 2, blocks // 2 + 5])
    flat[pages[2]] = 2.0 ** -4
    ks, vs = (rt.DeviceArray.of(flat) for _ in range(2))
    small = kv8.cache_of(rng, 4, kv, block, dim, ref.INT8)
    size = kv * dim * block
    for i, page in enumerate(pages):
        for d, a in ((dk, small[0]), (dv, small[1])):
            rt.check(rt.library().lh_copy_to_device(d.ptr + int(page) * size, np.ascontiguousarray(a[i]).ctypes.data, size))
    rows, length, path = 40, 160, [0, 5, 39]
    depth, seen = drafts.plan(drafts.random_tree(rng, rows, 4))
    q = rng.standard_normal((heads, rows, dim)).astype(np.float32)
    d = {"table": ints(rt, pages[None]), "lengths": ints(rt, [length]), "starts": ints(rt, [0, rows]), "rows": ints(rt, [rows])}
    dq, out, masks = rt.DeviceArray.of(q), rt.DeviceArray((rows, heads, dim), np.float32), rt.DeviceArray.of(drafts.packed(seen, 1))
    batch = rt.KvBatch(requests=1, tokens=rows, max_rows=rows, block=block, blocks=blocks, width=4, **{k: v.ptr for k, v in d.items()})
    cache = rt.Kv8(dk.ptr, dv.ptr, ks.ptr, vs.ptr, kv, dim, ref.INT8)
    rt.attention_kv8_tree(batch, cache, dq, heads, masks, out)
    own = np.array([[2.0 ** -5] * kv] * 4, np.float32)
    own[2] = 2.0 ** -4
    want, table = np.zeros((rows, heads, dim)), np.arange(4)[None]
    A = drafts.attention(q, small[0], small[1], own, own, table, [length], [0, rows], [rows], [seen], length - rows + depth, block, ref.INT8, 0, want)
    assert np.max(np.abs(out.numpy() - want)) <= kv8.bound(A, length, 127 * 2.0 ** -4)
    rt.kv8_compact(batch, [cache], ints(rt, path + [-1] * (rows - 3)), ints(rt, [3]))
    rt.synchronize()
    for d, i, transposed in ((dk, 0, False), (dv, 1, True)):
        codes, scales = small[i].copy(), own.copy()
        drafts.compact(codes, scales, table, [length], [0], [rows], np.array(path + [-1] * (rows - 3)), [3], block, ref.INT8, transposed)
        for j, page in enumerate(pages):
            got = np.empty_like(codes[j])
            rt.check(rt.library().lh_copy_to_host(got.ctypes.data, d.ptr + int(page) * size, size))
            assert np.array_equal(got, codes[j]), (i, j)

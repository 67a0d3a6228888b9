"""The entry points of drafted trees on the host: what they refuse, which kernels they launch, and the plain forms that
their tests compare with.

No kernel runs (fake_hip.py).
"""
from __future__ import annotations

import numpy as np
import pytest

from tests import drafts_reference as drafts
from tests import kv8_reference as ref
from tests.fake_hip import fake_hip  # noqa: F401  (fixture)
from tests.test_kv8_calls import BATCHES, CACHES, CALLS

TREE_CALLS = CALLS + '''
given = ("logits", "draft_logits", "ids", "parents", "temperatures", "accept", "sample", "path", "kept", "next")
def drafts(**changed): return rt.Drafts(**{"vocab": 100, **{k: buffer.ptr for k in given}, **changed})
def tree(b=None, parents=0, masks=0): return status(lib.lh_kv_tree(C.byref(b or batch()), buffer.ptr + parents, buffer.ptr + masks, None))
def attend_tree(b=None, c=None, q=0, heads=4, window=0, masks=0, out=0, workspace=None, bytes=0):
    return status(lib.lh_attention_kv8_tree(C.byref(b or batch()), C.byref(c or cache()), buffer.ptr + q, heads, window,
                                            (buffer.ptr + masks) or None, buffer.ptr + out, workspace, bytes, None))
def verify(b=None, d=None, workspace=None, bytes=0):
    return status(lib.lh_verify_drafts(C.byref(b or batch()), C.byref(d or drafts()), workspace, bytes, None))
def compact(b=None, caches=None, path=0, kept=0, layers=None):
    caches = [cache()] if caches is None else caches
    array = (rt.Kv8 * max(1, len(caches)))(*caches)
    return status(lib.lh_kv8_compact(C.byref(b or batch()), array, len(caches) if layers is None else layers, (buffer.ptr + path) or None,
                                     (buffer.ptr + kept) or None, None))
def keep(b=None, kept=0, lengths=0): return status(lib.lh_kv_keep(C.byref(b or batch()), (buffer.ptr + kept) or None, (buffer.ptr + lengths) or None, None))
'''


def refused(fake_hip, calls):
    results = fake_hip(TREE_CALLS + "result = [" + ", ".join(calls) + "]")
    for (code, message, launched), call in zip(results, calls):
        assert code == 1 and message.startswith("Leaf decoder: ") and launched == 0, (call, code, message)


def test_refused_batches_and_caches(fake_hip):  # noqa: F811
    refused(fake_hip, [f"{call}(batch({b}))" for b in BATCHES for call in ("tree", "attend_tree", "verify", "compact", "keep")] +
            [f"{call}(batch(max_rows=513))" for call in ("tree", "attend_tree", "verify", "compact")] +
            [f"attend_tree(c=cache({c}))" for c in CACHES] + [f"compact(caches=[cache(), cache({c})])" for c in CACHES])


def test_refused_arguments(fake_hip):  # noqa: F811
    refused(fake_hip, [f"tree(batch({n}=None))" for n in ("lengths", "starts", "rows", "positions")] +
            ["tree(parents=-buffer.ptr)", "tree(masks=-buffer.ptr)"] +
            [f"attend_tree(batch({n}=None))" for n in ("table", "lengths", "starts", "rows")] +
            ["attend_tree(batch(positions=None), window=5)", "attend_tree(masks=-buffer.ptr)", "attend_tree(heads=3)", "attend_tree(q=4)",
             "attend_tree(out=8)", "attend_tree(q=-buffer.ptr)", "attend_tree(out=-buffer.ptr)",
             "attend_tree(workspace=buffer.ptr + 8, bytes=1 << 20)", "attend_tree(batch(tokens=2**20), heads=130)"] +
            [f"verify(batch({n}=None))" for n in ("starts", "rows")] +
            [f"verify(d=drafts({n}=None))" for n in ("logits", "ids", "parents", "temperatures", "accept", "sample", "path", "kept", "next")] +
            ["verify(d=drafts(vocab=0))", "verify(d=drafts(vocab=2**30 + 1))", "verify(d=drafts(vocab=2**32 - 1))",
             "verify(workspace=buffer.ptr + 8, bytes=1 << 20)"] +
            [f"compact(batch({n}=None))" for n in ("table", "lengths", "starts", "rows")] +
            ["compact(path=-buffer.ptr)", "compact(kept=-buffer.ptr)", "compact(layers=0)", "compact(layers=65536)",
             "compact(caches=[cache(), cache(dim=32)])", "compact(caches=[cache(), cache(format=1)])", "compact(caches=[cache(), cache(kv_heads=1)])"] +
            [f"keep(batch({n}=None))" for n in ("table", "lengths", "rows", "free_blocks", "free_count", "free_left")] +
            ["keep(kept=-buffer.ptr)", "keep(lengths=-buffer.ptr)"])


def test_accepted_calls(fake_hip):  # noqa: F811
    results = fake_hip(TREE_CALLS + '''
result = [tree(), tree(batch(max_rows=512, tokens=600)), attend_tree(), attend_tree(batch(positions=None)), attend_tree(window=2**32 - 1),
          attend_tree(c=cache(dim=256, format=1)), verify(), verify(d=drafts(draft_logits=None)), verify(batch(lengths=None, table=None)),
          compact(), compact(caches=[cache()] * 33), compact(batch(requests=4000, tokens=4000)), keep(), keep(batch(max_rows=5000, requests=4000)),
          attend_tree(batch(max_rows=512, tokens=2))]
''')
    assert all(code == 0 and launched >= 1 for code, _, launched in results), results
    assert results[10][2] == 2                              # 32 layers a launch


def test_batches_that_are_null(fake_hip):  # noqa: F811
    results = fake_hip(TREE_CALLS + '''
b, c, d, p = C.byref(batch()), C.byref(cache()), C.byref(drafts()), buffer.ptr
result = [status(s) for s in (lib.lh_kv_tree(None, p, p, None), lib.lh_attention_kv8_tree(None, c, p, 4, 0, p, p, None, 0, None),
          lib.lh_attention_kv8_tree(b, None, p, 4, 0, p, p, None, 0, None), lib.lh_verify_drafts(None, d, None, 0, None),
          lib.lh_verify_drafts(b, None, None, 0, None), lib.lh_verify_drafts_workspace(b, d, None),
          lib.lh_kv8_compact(None, c, 1, p, p, None), lib.lh_kv8_compact(b, None, 1, p, p, None), lib.lh_kv_keep(None, p, p, None))]
''')
    assert all(code == 1 and launched == 0 for code, _, launched in results), results


@pytest.mark.parametrize("sizes,heads,kernels", [
    ("requests=64, tokens=512, max_rows=8, width=64", 4, ["few_kernel", "tree_merge"]),        # 16 rows of a KV head
    ("requests=64, tokens=512, max_rows=8, width=8", 4, ["few_kernel"]),                       # too short to be parted
    ("requests=64, tokens=512, max_rows=9, width=64", 4, ["tree_kernel", "tree_merge"]),
    ("requests=64, tokens=512, max_rows=9, width=20", 4, ["tree_kernel"]),
    ("requests=51, tokens=300, max_rows=200, width=64", 4, ["tree_kernel", "tree_merge"]),
    ("requests=64, tokens=64, max_rows=1, width=64", 34, ["tree_kernel", "tree_merge"])])      # groups of 17
def test_attention_routes(fake_hip, sizes, heads, kernels):  # noqa: F811
    launched = fake_hip(TREE_CALLS + f"""
b, code = batch({sizes}), None
code = lib.lh_attention_kv8_tree(C.byref(b), C.byref(cache()), buffer.ptr, {heads}, 0, buffer.ptr, buffer.ptr, None, 0, None)
result = [code, kernels()]
""")
    assert launched[0] == 0 and len(launched[1]) == len(kernels), launched
    assert all(f"attention_kv8_{name}" in k for name, k in zip(kernels, launched[1])), launched


@pytest.mark.parametrize("sizes,vocab,draft,kernels", [
    ("requests=1, tokens=5, max_rows=5", 32000, True, ["verify_rows", "verify_kernel"]),       # few logits: every row ahead
    ("requests=64, tokens=512, max_rows=8", 32000, True, ["empty_slots", "verify_kernel"]),
    ("requests=64, tokens=64, max_rows=1", 32000, False, ["empty_slots", "verify_kernel"]),    # no drafts: sampling alone
    ("requests=300, tokens=600, max_rows=512", 20000, False, ["verify_kernel"]),               # a workgroup for a request
    ("requests=1, tokens=1, max_rows=1", 2048, False, ["verify_kernel"]),
    ("requests=300, tokens=600, max_rows=512", 2000, False, ["verify_kernel"])])               # mostly rows that no request has
def test_verification_routes(fake_hip, sizes, vocab, draft, kernels):  # noqa: F811
    launched = fake_hip(TREE_CALLS + f"""
b, d = batch({sizes}), drafts(vocab={vocab}, draft_logits={"buffer.ptr" if draft else None})
n = C.c_size_t()
result = [lib.lh_verify_drafts_workspace(C.byref(b), C.byref(d), C.byref(n)), n.value, lib.lh_verify_drafts(C.byref(b), C.byref(d), None, 0, None), kernels()]
""")
    assert launched[0] == launched[2] == 0 and len(launched[3]) == len(kernels), launched
    assert all(name in k for name, k in zip(kernels, launched[3])), launched
    assert (launched[1] > 0) == (len(kernels) > 1)


def test_workspace_does_not_depend_on_lengths(fake_hip):  # noqa: F811
    sizes, error = fake_hip(TREE_CALLS + """
n, result = C.c_size_t(), []
for width in (64, 4096, 2**20):
    assert lib.lh_attention_kv8_tree_workspace(C.byref(batch(requests=64, tokens=512, max_rows=9, width=width)), C.byref(cache(keys=None, values=None)), 8, C.byref(n)) == 0
    result.append(n.value)
result = [result, lib.lh_attention_kv8_tree_workspace(C.byref(batch()), C.byref(cache()), 8, None)]
""")
    assert sizes[1] == sizes[2] <= 64 << 20 and sizes[0] <= sizes[1] and error == 1


# ---- the plain forms themselves
def test_plans():
    depth, seen = drafts.plan([-1, 0, 0, 1, 7, 3])          # row 4's parent is no earlier row
    assert list(depth) == [0, 1, 1, 2, 0, 3]
    assert [list(np.nonzero(s)[0]) for s in seen] == [[0], [0, 1], [0, 2], [0, 1, 3], [4], [0, 1, 3, 5]]
    assert drafts.packed(seen, 1)[:, 0].tolist() == [1, 3, 5, 11, 16, 43]


@pytest.mark.parametrize("with_draft", [False, True])
def test_verification_keeps_the_distribution(with_draft):
    # of two drafted tokens behind one row (drawn from q, or fixed) and random numbers: the token that follows the row, a kept
    # child's or the one behind, is distributed as p; 20000 trials, five standard deviations
    rng = np.random.default_rng(3)
    vocab, trials = 5, 20000
    logits, draft = rng.standard_normal((3, vocab)), rng.standard_normal((3, vocab))
    p, q = drafts.softmax(logits[0], 0.8), drafts.softmax(draft[0], 0.8)
    counts = np.zeros(vocab)
    for _ in range(trials):
        ids = np.concatenate([[0], rng.choice(vocab, 2, p=q) if with_draft else [3, 1]])
        path, following = drafts.verify(logits, draft if with_draft else None, ids, [-1, 0, 0], 0.8, rng.random(3), rng.random())
        counts[ids[path[1]] if len(path) > 1 else following] += 1
    assert (np.abs(counts - trials * p) < 5 * np.sqrt(trials * p * (1 - p))).all()


def test_compaction_moves_rows_and_scales():
    # blocks of 4: cached 0..1, rows at 2..6 of which 0, 2 and 4 stand: 2 <- 2, 3 <- 4, 4 <- 6
    codes, scales = np.zeros((2, 1, 4, 1), np.uint8), np.array([[1.0], [2.0]], np.float32)
    codes[0, 0, :, 0], codes[1, 0, :, 0] = (10, 11, 12, 13), (24, 25, 26, 27)
    drafts.compact(codes, scales, np.array([[0, 1]]), [7], [0], [5], np.array([0, 2, 4, -1, -1]), [3], 4, ref.INT8, False)
    assert list(codes[0, 0, :, 0]) == [5, 6, 6, 24] and list(codes[1, 0, :, 0]) == [26, 25, 26, 27]
    assert scales.tolist() == [[2.0], [2.0]]                 # 11 / 2 = 5.5 and 13 / 2 to the even neighbour


def test_keeping_gives_blocks_back():
    table = np.array([[3, 4, 5], [6, 7, 8]])
    lengths, stack, count = drafts.keep([10, 9], [6, 4], [1, 4], table, np.array([9, 0, 0, 0]), 1, 4, 10)
    assert list(lengths) == [5, 9] and count == 2 and list(stack[:2]) == [9, 5]

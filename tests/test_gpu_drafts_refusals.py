"""Verification after many refused children of one row, whose refusals leave next to nothing of the target's distribution.

What is left is then of the size of its own rounding, so which token follows is open; but one does, from the
distribution (include/leafhip.h: next).
"""
from __future__ import annotations

import numpy as np
import pytest

from tests import drafts_reference as drafts
from tests.test_gpu_drafts import check_verify, rt, verify_on_gpu  # noqa: F401  (rt: fixture)

pytestmark = pytest.mark.gpu


def refused_case(rng, requests, rows, vocab, with_draft):
    """Stars: children of row 0 with a token that the target likes less than the draft does, until all that is left is one
    token of which the target has 0.32 and the draft 0.25: a refusal takes that share of it.  Neither has most of
    it: its neighbour and a token far away have more."""
    counts = rng.integers(rows // 2, rows + 1, requests)
    starts, tokens = np.concatenate([[0], np.cumsum(counts)]), int(counts.sum())
    logits = rng.standard_normal((tokens, vocab)).astype(np.float32)
    draft = (logits + 0.05 * rng.standard_normal((tokens, vocab))).astype(np.float32)
    parents, ids, temperatures = np.zeros(tokens, int), np.zeros(tokens, int), rng.uniform(0.5, 1.5, requests).astype(np.float32)
    for r, t in enumerate(starts[:-1]):
        parents[t], x = -1, int(rng.integers(vocab - 1))
        three = [x, x + 1, (x + vocab // 2) % vocab]
        for row, shares in ((logits[t], (0.32, 0.33, 0.34)), (draft[t], (0.25, 0.35, 0.36))):
            others = np.delete(row, three).astype(np.float64) / temperatures[r]
            row[three] = temperatures[r] * (np.log(np.exp(others).sum()) + np.log(np.array(shares) / (1 - sum(shares))))
        p, q = (drafts.softmax(x[t], temperatures[r]) for x in (logits, draft))
        ids[t + 1:starts[r + 1]] = int(np.argmin(p / q)) if with_draft else rng.integers(vocab, size=counts[r] - 1)
    return dict(logits=logits, draft_logits=draft if with_draft else None, ids=ids, parents=parents, temperatures=temperatures,
                accept=np.full(tokens, 1 - 2.0 ** -24, np.float32), sample=rng.random(requests).astype(np.float32),
                starts=starts, rows=counts)


# a segment for a request with its weights in LDS, sixteen of them, and (few logits) rows measured ahead
@pytest.mark.parametrize("requests,rows,vocab", [(120, 150, 2000), (6, 120, 32000), (2, 500, 10000), (3, 90, 5000)])
def test_a_token_follows_whatever_is_left(rt, requests, rows, vocab):  # noqa: F811
    rng = np.random.default_rng(requests + vocab)
    c = refused_case(rng, requests, rows, vocab, True)
    path, kept, following = verify_on_gpu(rt, c)              # (preset to -7)
    assert (kept == 1).all() and (path[c["starts"][:-1]] == 0).all()
    assert ((following >= 0) & (following < vocab)).all(), np.argwhere(following < 0)[:, 0]


@pytest.mark.parametrize("with_draft", [False, True])
@pytest.mark.parametrize("requests,rows,vocab", [(120, 30, 2000), (10, 30, 32000), (3, 30, 5000)])
def test_the_token_behind_some_refusals(rt, requests, rows, vocab, with_draft):  # noqa: F811
    # 0.1 times 0.75^29 and more are left: more than enough for the plain form's token
    rng = np.random.default_rng(requests + vocab + 1)
    kept, _ = check_verify(rt, refused_case(rng, requests, rows, vocab, with_draft))
    assert (kept == 1).all()

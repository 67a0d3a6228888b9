"""Plain 64-bit forms of the operators of drafted trees (include/leafhip.h: lh_kv_tree to lh_kv_keep)."""
from __future__ import annotations

import numpy as np

from tests import kv8_reference as ref


def random_tree(rng, rows, reach):
    """Parents of a tree whose rows hang on one of the `reach` rows before them (1: a chain)."""
    return np.array([-1] + [int(rng.integers(max(0, i - reach), i)) for i in range(1, rows)])


def plan(parents):
    """(depths, ancestors [rows, rows]); a parent that is no earlier row is the cached text."""
    n = len(parents)
    depth, seen = np.zeros(n, int), np.eye(n, dtype=bool)
    for i, p in enumerate(parents):
        if 0 <= p < i:
            depth[i], seen[i] = depth[p] + 1, seen[i] | seen[p]
    return depth, seen


def packed(seen, words):
    """[rows, rows] truth values to masks [rows, words]."""
    masks = np.zeros((len(seen), words), np.uint64)
    for j in range(seen.shape[1]):
        masks[:, j // 64] |= seen[:, j].astype(np.uint64) << np.uint64(j % 64)
    return masks


def attention(q, keys, values, key_scales, value_scales, table, lengths, starts, rows, seen, positions, block, form, window, out):
    """kv8_reference.attention of trees: seen[r] [rows, rows] are request r's ancestors, positions [tokens]."""
    heads, _, dim = q.shape
    group, largest, blocks = heads // keys.shape[1], 0.0, len(keys)
    for r in range(len(rows)):
        if rows[r] <= 0 or lengths[r] < rows[r]:
            continue
        pages = table[r, :-(-lengths[r] // block)]
        known = (pages >= 0) & (pages < blocks)
        at = np.where(known, pages, 0)
        before = lengths[r] - rows[r]
        own = positions[starts[r]:starts[r] + rows[r]]
        for kvh in range(keys.shape[1]):
            ks = np.where(known, key_scales[at, kvh], np.nan).astype(np.float64)
            vs = np.where(known, value_scales[at, kvh], np.nan).astype(np.float64)
            k = (ref.decode(keys[at, kvh], form) * ks[:, None, None]).reshape(-1, dim)[:lengths[r]]
            v = (ref.decode(values[at, kvh], form) * vs[:, None, None]).transpose(0, 2, 1).reshape(-1, dim)[:lengths[r]]
            for i in range(rows[r]):
                visible = np.concatenate([np.ones(before, bool), seen[r][i]])
                if window:
                    stand = max(int(own[i]), before)
                    visible &= np.concatenate([np.arange(before), own]) > stand - window
                for h in range(kvh * group, (kvh + 1) * group):
                    if not visible.any():
                        out[starts[r] + i, h] = 0.0
                        continue
                    x = q[h, starts[r] + i].astype(np.float64)
                    with np.errstate(invalid="ignore"):
                        s = k[visible] @ x / np.sqrt(dim)
                    if not np.isfinite(s).all() or not np.isfinite(v[visible]).all():
                        out[starts[r] + i, h] = np.nan
                        continue
                    p = np.exp(s - s.max())
                    out[starts[r] + i, h] = (p / p.sum()) @ v[visible]
                    largest = max(largest, float((np.abs(k[visible]) @ np.abs(x)).max()) / np.sqrt(dim))
    return largest


def softmax(logits, temperature):
    """In 64 bits; None where there is no distribution."""
    x = logits.astype(np.float64)
    if np.isnan(x).any() or (x == np.inf).any() or (x == -np.inf).all() or not 0 < temperature < np.inf:
        return None
    p = np.exp((x - x.max()) / np.float64(temperature))
    return p / p.sum()


def verify(logits, draft, ids, parents, temperature, accept, sample):
    """One request: (path, next).  logits [rows, vocab]; draft the same or None."""
    path, row, i, vocab = [0], 0, 1, logits.shape[1]
    r = q = None

    def first_largest():
        x = logits[row]
        return None if np.isnan(x).any() or (x == np.inf).any() or (x == -np.inf).all() else int(np.argmax(x))
    while i < len(parents):
        if parents[i] != row:
            i += 1
            continue
        x, taken = int(ids[i]), accept[i] < 0
        if not taken:
            if temperature == 0:
                best = first_largest()
                if best is None:
                    return path, -1
                taken = x == best
            else:
                if r is None:
                    r = softmax(logits[row], temperature)
                    if r is None:
                        return path, -1
                if 0 <= x < vocab:
                    if draft is not None and q is None:
                        q = softmax(draft[row], temperature)
                        if q is None:
                            return path, -1
                    u, S = np.float64(accept[i]), r.sum()
                    taken = u * S * (1.0 if q is None else q[x]) < r[x]
                    if not taken and q is None:
                        r[x] = 0.0
                    elif not taken:
                        r = np.maximum(r - S * q, 0.0)
        if taken:
            path.append(i)
            row, r, q = i, None, None
        i += 1
    if temperature == 0:
        best = first_largest()
        return path, -1 if best is None else best
    p = softmax(logits[row], temperature)
    if p is None:
        return path, -1
    r = p if r is None or not r.sum() > 0 else r
    goal = np.float64(min(max(sample, 0.0), 1.0)) * r.sum()
    passed = np.nonzero((np.cumsum(r) > goal) & (r > 0))[0]
    return path, int(passed[0]) if len(passed) else int(np.nonzero(r > 0)[0][-1])


def compact(codes, scales, table, lengths, starts, rows, path, kept, block, form, transposed):
    """The kept rows of one layer's keys or values moved together, in place."""
    blocks, was, scale_was = len(codes), codes.copy(), scales.copy()
    for r in range(len(rows)):
        own = np.asarray(path[starts[r]:starts[r] + kept[r]]) if rows[r] > 0 else np.zeros(0, int)
        if not 0 < kept[r] <= rows[r] or own[0] < 0 or own[-1] >= rows[r] or (np.diff(own) <= 0).any():
            continue
        before = lengths[r] - rows[r]
        comes = {}
        for k, place in enumerate(own):
            comes.setdefault((before + k) // block, []).append((before + k, before + int(place)))
        for entry, moves in comes.items():
            to = table[r, entry]
            if not 0 <= to < blocks or all(a == b for a, b in moves):
                continue
            moves = [(p, p) for p in range(entry * block, min(before, (entry + 1) * block))] + moves
            moves = [(a, table[r, b // block], b) for a, b in moves if 0 <= table[r, b // block] < blocks]
            for h in range(codes.shape[1]):
                given = [scale_was[page, h] for _, page, _ in moves]
                fine = all(0 <= s < np.inf for s in given)
                scale = np.float32(max(given)) if fine else np.float32(np.nan)
                for a, page, b in moves:
                    source, held = (x[:, :].T if transposed else x for x in (was[page, h], codes[to, h]))
                    old = scale_was[page, h]
                    held[a % block] = source[b % block] if not fine or old == scale else \
                        ref.encode(ref.decode(source[b % block], form) * np.float64(old) / np.float64(scale), form)
                scales[to, h] = scale


def keep(lengths, rows, kept, table, stack, count, block, blocks):
    """(lengths, stack, count) after a step of which kept rows stand."""
    lengths, stack = np.array(lengths), stack.copy()
    for r in range(len(rows)):
        if not 0 < rows[r] <= lengths[r] or not 0 <= kept[r] <= rows[r]:
            continue
        after = lengths[r] - rows[r] + kept[r]
        for entry in range(-(-after // block), -(-lengths[r] // block)):
            if count < blocks:
                stack[count], count = table[r, entry], count + 1
        lengths[r] = after
    return lengths, stack, count

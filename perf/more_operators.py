"""The operators of drafted trees over the 8-bit KV cache: what is timed, and their plain forms.

A program that serves several requests lets a small model draft some tokens for
each, as a tree, and checks all of them in one step of the large model:

* ``tree``: positions and ancestor masks of the step's rows, from their parents;
* ``attend``: attention of the rows over their requests' blocks and their own ancestors;
* ``verify``: which drafted tokens stand, from both models' logits and given random numbers, and the token behind them;
* ``keep``: the kept rows moved together in every layer's cache, lengths and blocks put right.

Head layouts, vocabularies and layer counts are those of the presets in
``leaf_amd/models.py``, and heads of 128. ``run`` computes the operators from
elementary torch operations, or with ``own`` calls the library.
"""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import torch

own = False

# (heads, kv_heads, dim) of the presets, of heads of 128 and of 80.
LAYOUTS = ((32, 4, 64), (14, 2, 64), (15, 5, 64), (12, 12, 64), (32, 8, 128), (8, 2, 80))
VOCABULARIES = (32000, 49152, 50257, 151936)
INT8, E4M3 = 0, 1
CHAIN = 1                                            # a tree's branching: every row the child of the one before it


# ------------------------------------------------------------------- cases ---
def _tree(requests, rows, branch, longest=3000, mix=1):
    return {"kind": "tree", "requests": requests, "rows": rows, "branch": branch, "shortest": 0, "longest": longest, "mix": mix}


def _attend(requests, rows, branch, shortest, longest, layout, block, form, window=0, mix=1):
    heads, kv_heads, dim = layout
    return {"kind": "attend", "requests": requests, "rows": rows, "branch": branch, "shortest": shortest,
            "longest": longest, "heads": heads, "kv_heads": kv_heads, "dim": dim, "block": block, "form": form,
            "window": window, "mix": mix}


def _verify(requests, rows, branch, vocab, draft, greedy=False, mix=1):
    return {"kind": "verify", "requests": requests, "rows": rows, "branch": branch, "shortest": 0, "longest": 0,
            "vocab": vocab, "draft": draft, "greedy": greedy, "mix": mix}


def _keep(requests, rows, branch, layers, layout, block, form, mix=1):
    _, kv_heads, dim = layout
    return {"kind": "keep", "requests": requests, "rows": rows, "branch": branch, "shortest": 0, "longest": block - 1,
            "layers": layers, "kv_heads": kv_heads, "dim": dim, "block": block, "form": form, "mix": mix}


def listed():
    cases = {
        # A small server's step with eight drafted rows for each of 24 requests: the smallest call.
        "tree_step": _tree(24, 8, 2),
        # A large server's step of wide trees.
        "tree_wide": _tree(250, 64, 3),
        # One conversation at a context of 4095 tokens, a tree of 26 rows.
        "attend_single": _attend(1, 26, 3, 4095, 4095, (14, 2, 64), 64, INT8),
        # 64 requests at ragged contexts, seven drafted tokens each, heads of 128 grouped by four.
        "attend_batch": _attend(64, 8, CHAIN, 200, 4096, (32, 8, 128), 64, INT8),
        # Wide trees for 16 requests at long contexts, 8-bit floating point, heads grouped by eight.
        "attend_wide": _attend(16, 64, 3, 500, 8000, (32, 4, 64), 32, E4M3),
        # 40 requests in small blocks with a sliding window, an odd number of rows, heads grouped by three.
        "attend_window": _attend(40, 13, 2, 30, 2000, (15, 5, 64), 16, E4M3, window=1024),
        # One conversation: a chain of four drafted tokens, sampled.
        "verify_single": _verify(1, 5, CHAIN, 32000, True),
        # 64 requests, small trees, both models' logits.
        "verify_batch": _verify(64, 8, 2, 32000, True),
        # Wide trees over the largest vocabulary, drafts without probabilities.
        "verify_wide": _verify(16, 26, 3, 151936, False),
        # A batch that decodes greedily.
        "verify_greedy": _verify(100, 4, CHAIN, 49152, False, greedy=True),
        # The kept rows of 64 requests in 22 layers.
        "keep_batch": _keep(64, 8, 2, 22, (32, 4, 64), 16, INT8),
        # Wide trees, 24 layers, larger blocks, 8-bit floating point.
        "keep_wide": _keep(16, 64, 3, 24, (14, 2, 64), 64, E4M3),
    }
    return [dict(case, name=name) for name, case in cases.items()]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("tree", "attend", "attend", "verify", "verify", "keep"))
    mix, branch = rng.randint(2, 1 << 20), rng.choice((CHAIN, 2, 3, 4))
    layout, block, form = rng.choice(LAYOUTS), rng.choice((16, 32, 64, 128)), rng.choice((INT8, E4M3))
    if kind == "tree":
        requests = _log_int(rng, 1, 500)
        return _tree(requests, _log_int(rng, 2, min(300, 16000 // requests)), branch, mix=mix)
    if kind == "attend":
        heads, kv_heads, dim = layout
        rows, longest = _log_int(rng, 1, 64), _log_int(rng, 20, 8000)
        most = min(2.0e8 / (kv_heads * dim * longest), 2.5e8 / (heads * rows * longest))
        requests = min(_log_int(rng, 1, 100), max(1, int(most)))
        return _attend(requests, rows, branch, max(1, longest // 20), longest, layout, block, form,
                       rng.choice((0, 0, 0, 500)), mix)
    if kind == "verify":
        vocab, rows = rng.choice(VOCABULARIES), _log_int(rng, 1, 40)
        requests = min(_log_int(rng, 1, 120), max(1, int(6.0e7 / (vocab * rows))))
        return _verify(requests, rows, branch, vocab, rng.random() < 0.6, rng.random() < 0.2, mix)
    rows, requests = _log_int(rng, 2, 64), _log_int(rng, 1, 64)
    layers = rng.randint(1, max(1, min(32, int(3.0e7 / (requests * (rows + block) * layout[1] * layout[2])))))
    return _keep(requests, rows, branch, layers, layout, block, form, mix)


def _plan(case):
    """(cached, rows, parents): ragged requests and trees, the same for every seed, so that the work is."""
    r, n, most = np.random.RandomState(case["mix"]), case["requests"], case["rows"]
    cached = r.randint(case["shortest"], case["longest"] + 1, n)
    rows = r.randint(max(1, most - most // 3), most + 1, n)
    rows[r.randint(n)] = most
    parents = []
    for count in rows:
        if case["branch"] == CHAIN:
            tree = np.arange(-1, count - 1)
        else:                                        # level by level, about `branch` children a row
            i = np.arange(count)
            tree = np.minimum(((i - 1) / case["branch"] * r.uniform(0.6, 1.4, count)).astype(int), i - 1)
            tree[0] = -1
        parents.append(tree)
    return cached, rows, parents


def _depths(parents):
    depth = np.zeros(len(parents), int)
    for i in range(1, len(parents)):
        depth[i] = depth[parents[i]] + 1
    return depth


def _ancestors(parents):
    """[rows, rows]: whether row j is row i or one of its ancestors."""
    seen = np.eye(len(parents), dtype=bool)
    for i, parent in enumerate(parents):
        if parent >= 0:
            seen[i] |= seen[parent]
    return seen


def _paths(case):
    """A kept path of each request: down the tree with three chances in four a level."""
    _, rows, parents = _plan(case)
    r = np.random.RandomState(case["mix"] + 1)
    paths = []
    for tree in parents:
        path = [0]
        while True:
            children = np.nonzero(tree == path[-1])[0]
            if not len(children) or r.rand() > 0.75:
                break
            path.append(int(r.choice(children)))
        paths.append(path)
    return paths


def _blocks_of(tokens, block):
    return -(-tokens // block)


# ------------------------------------------------------------------ inputs ---
def _ints(a):
    return torch.as_tensor(np.ascontiguousarray(a), dtype=torch.int32, device="cuda")


def _codes(gen, shape, form):
    """Codes of N(0, 1) values under scales that differ from block to block: shape is [..., blocks, kv_heads, a, b]."""
    x = torch.randn(shape, generator=gen, device="cuda")
    scale = torch.exp(0.3 * torch.randn(shape[:-2], generator=gen, device="cuda")) * (4.0 / 127 if form == INT8 else 2.0 ** -6)
    if form == INT8:
        return (32 * x).round_().clamp_(-127, 127).to(torch.int8), scale
    return (64 * x).clamp_(-448, 448).to(torch.float8_e4m3fn), torch.exp2(torch.round(torch.log2(scale)))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    cached, rows, parents = _plan(case)
    n, tokens, most = case["requests"], int(rows.sum()), int(rows.max())
    starts = np.concatenate([[0], np.cumsum(rows)])
    s = {"case": case, "tokens": tokens, "max_rows": most, "width": 1, "blocks": 1, "block": case.get("block", 16),
         "starts": _ints(starts), "rows": _ints(rows), "lengths": _ints(cached + rows),
         "parents": _ints(np.concatenate(parents)),
         "request": torch.as_tensor(np.repeat(np.arange(n), rows), device="cuda")}
    if case["kind"] == "tree":
        # (the masks say nothing of the cache: a table of any width does)
        s["width"] = _blocks_of(case["longest"] + most, s["block"])
        s["positions"] = torch.full((tokens,), -1, dtype=torch.int32, device="cuda")
        s["masks"] = torch.zeros(tokens, _blocks_of(most, 64), dtype=torch.int64, device="cuda")
        # (which tree the program drafted differs from step to step: a row's children may be its parent's too)
        if case["branch"] != CHAIN:
            r = np.random.RandomState(seed % (1 << 31))
            parents = [np.where((r.rand(len(tree)) < 0.2) & (tree > 0), tree[np.maximum(tree, 0)], tree) for tree in parents]
            s["parents"] = _ints(np.concatenate(parents))
    elif case["kind"] == "verify":
        _prepare_verify(case, gen, s)
    else:
        _prepare_blocks(case, gen, s, cached, rows)
        if case["kind"] == "attend":
            s["positions"] = _ints(np.concatenate([c + _depths(tree) for c, tree in zip(cached, parents)]))
            s["masks"] = torch.as_tensor(_packed(parents, _blocks_of(most, 64)), device="cuda")
            s["q"] = torch.randn(case["heads"], tokens, case["dim"], generator=gen, device="cuda")
            s["out"] = torch.empty(tokens, case["heads"] * case["dim"], device="cuda")
        else:
            path, kept = np.full(tokens, -1), np.zeros(n)
            for r, one in enumerate(_paths(case)):
                path[starts[r]:starts[r] + len(one)], kept[r] = one, len(one)
            s["path"], s["kept"], s["after"] = _ints(path), _ints(kept), _ints(np.zeros(n))
    if own:
        _describe(s)
    return s


def _packed(parents, words):
    """The ancestor masks of all rows: bit j % 64 of word j / 64."""
    masks = np.zeros((sum(map(len, parents)), words), np.uint64)
    first = 0
    for tree in parents:
        seen = _ancestors(tree)
        for j in range(len(tree)):
            masks[first:first + len(tree), j // 64] |= seen[:, j].astype(np.uint64) << np.uint64(j % 64)
        first += len(tree)
    return masks.view(np.int64)


def _prepare_verify(case, gen, s):
    tokens, vocab, n = s["tokens"], case["vocab"], case["requests"]
    s["logits"] = 3.5 * torch.randn(tokens, vocab, generator=gen, device="cuda")
    draft = s["logits"] + 0.6 * torch.randn(tokens, vocab, generator=gen, device="cuda")
    s["temperatures"] = torch.zeros(n, device="cuda") if case["greedy"] else \
        0.6 + 0.6 * torch.rand(n, generator=gen, device="cuda")
    # a drafted token is drawn from its parent's row of the draft's logits
    warm = s["temperatures"][s["request"]]
    s["ids"] = torch.randint(0, vocab, (tokens,), generator=gen, device="cuda", dtype=torch.int32)
    parent = s["starts"].long()[s["request"]] + s["parents"]
    for first in range(0, tokens, 256):
        some = torch.arange(first, min(first + 256, tokens), device="cuda")
        uniform = torch.rand(len(some), vocab, generator=gen, device="cuda").clamp_(1e-9, 1 - 1e-7)
        noise = uniform.log_().neg_().log_().neg_().mul_(warm[some, None])
        token = (draft[parent[some].clamp(min=0)] + noise).argmax(1).int()
        s["ids"][some] = torch.where(s["parents"][some] >= 0, token, s["ids"][some])
    s["draft"] = draft if case["draft"] else None
    s["accept"] = torch.rand(tokens, generator=gen, device="cuda")
    s["sample"] = torch.rand(n, generator=gen, device="cuda")
    s["path"], s["kept"], s["next"] = (_ints(np.zeros(size)) for size in (tokens, n, n))


def _prepare_blocks(case, gen, s, cached, rows):
    """A step's tables as an earlier call has left them, over pools that hold the blocks of all requests."""
    block, kv, dim = case["block"], case["kv_heads"], case["dim"]
    held = _blocks_of(cached + rows, block)
    blocks, width = int(held.sum()), int(held.max())
    order = torch.randperm(blocks, generator=gen, device="cuda").int()
    entry = torch.arange(width, device="cuda")
    first = _ints(np.cumsum(held) - held)
    table = torch.where(entry < _ints(held)[:, None], order[(first[:, None] + entry).clamp(max=blocks - 1)], -1)
    layers = (case["layers"],) if case["kind"] == "keep" else ()
    s["table"], s["blocks"], s["width"] = table.int().contiguous(), blocks, width
    s["keys"], s["key_scales"] = _codes(gen, layers + (blocks, kv, block, dim), case["form"])
    s["values"], s["value_scales"] = _codes(gen, layers + (blocks, kv, dim, block), case["form"])
    s["stack"], s["count"], s["left"] = _ints(np.full(blocks, -1)), _ints([0]), _ints([0])


def _describe(s):
    """The library's descriptions of the batch and its caches, which a program keeps from step to step."""
    from leaf_amd import runtime
    case = s["case"]

    def at(name):
        return s[name].data_ptr() if s.get(name) is not None else None
    s["batch"] = runtime.KvBatch(
        requests=case["requests"], tokens=s["tokens"], max_rows=s["max_rows"], block=s["block"], blocks=s["blocks"],
        width=s["width"], free_blocks=at("stack"), free_count=at("count"), free_left=at("left"), table=at("table"),
        lengths=at("lengths"), starts=at("starts"), rows=at("rows"), positions=at("positions"))
    if "keys" in s:
        layers = case.get("layers", 1)
        s["caches"] = (runtime.Kv8 * layers)()
        for i in range(layers):
            arrays = (s[k][i] if "layers" in case else s[k] for k in ("keys", "values", "key_scales", "value_scales"))
            s["caches"][i] = runtime.Kv8(*(a.data_ptr() for a in arrays), case["kv_heads"], case["dim"], case["form"])
    if case["kind"] == "verify":
        s["drafts"] = runtime.Drafts(
            vocab=case["vocab"], logits=at("logits"), draft_logits=at("draft"), ids=at("ids"), parents=at("parents"),
            temperatures=at("temperatures"), accept=at("accept"), sample=at("sample"), path=at("path"), kept=at("kept"),
            next=at("next"))
    s["lib"], s["check"] = runtime.library(), runtime.check


# -------------------------------------------------------------------- runs ---
def run(state):
    return globals()[("_own_" if own else "_plain_") + state["case"]["kind"]](state)


def _own_tree(s):
    s["check"](s["lib"].lh_kv_tree(C.byref(s["batch"]), s["parents"].data_ptr(), s["masks"].data_ptr(), None))
    return {"positions": s["positions"], "masks": s["masks"]}


def _own_attend(s):
    case = s["case"]
    s["check"](s["lib"].lh_attention_kv8_tree(C.byref(s["batch"]), s["caches"], s["q"].data_ptr(), case["heads"],
                                              case["window"], s["masks"].data_ptr(), s["out"].data_ptr(), None, 0, None))
    return s["out"]


def _own_verify(s):
    s["check"](s["lib"].lh_verify_drafts(C.byref(s["batch"]), C.byref(s["drafts"]), None, 0, None))
    return {"path": s["path"], "kept": s["kept"], "next": s["next"]}


def _own_keep(s):
    lib, check, kept = s["lib"], s["check"], s["kept"].data_ptr()
    check(lib.lh_kv8_compact(C.byref(s["batch"]), s["caches"], s["case"]["layers"], s["path"].data_ptr(), kept, None))
    check(lib.lh_kv_keep(C.byref(s["batch"]), kept, s["after"].data_ptr(), None))
    return _kept(s, s["after"], s["stack"], s["left"])


def _values_of(codes, scales):
    """What codes stand for."""
    if codes.dtype == torch.int8:
        return codes * scales[..., None, None]
    return codes.float().mul_(scales[..., None, None])


def _kept(s, lengths, stack, left):
    return {"keys": _values_of(s["keys"], s["key_scales"]), "values": _values_of(s["values"], s["value_scales"]),
            "key_scales": s["key_scales"], "value_scales": s["value_scales"], "lengths": lengths, "stack": stack, "left": left}


def _plain_tree(s):
    n, most, words = s["case"]["requests"], s["max_rows"], s["masks"].shape[1]
    starts, rows, row = s["starts"].long()[:-1], s["rows"].long(), torch.arange(most, device="cuda")
    token = (starts[:, None] + row).clamp(max=s["tokens"] - 1)
    parent = torch.where(row < rows[:, None], s["parents"].long()[token], -1)
    # ancestors over 1, 2, 4.. generations
    seen = (row[:, None] == row) | (row == parent[:, :, None])
    for _ in range(max(1, (most - 1).bit_length())):
        seen = torch.matmul(seen.float(), seen.float()) > 0
    depth = seen.sum(-1) - 1
    bits = torch.nn.functional.pad(seen, (0, 64 * words - most)).view(n, most, words, 64)
    masks = (bits.long() << torch.arange(64, device="cuda")).sum(-1)
    index = torch.arange(s["tokens"], device="cuda") - starts[s["request"]]
    base = (s["lengths"].long() - rows)[s["request"]]
    return {"positions": (base + depth[s["request"], index]).int(), "masks": masks[s["request"], index]}


def _plain_attend(s):
    case = s["case"]
    heads, kv, dim, n, most = case["heads"], case["kv_heads"], case["dim"], case["requests"], s["max_rows"]
    group = heads // kv
    table = s["table"].long().clamp(min=0)
    keys = s["keys"].float()[table] * s["key_scales"][table][..., None, None]              # [n, width, kv, block, dim]
    values = s["values"].float()[table] * s["value_scales"][table][..., None, None]        # [n, width, kv, dim, block]
    keys = keys.permute(0, 2, 1, 3, 4).reshape(n, kv, -1, dim)
    values = values.permute(0, 2, 1, 4, 3).reshape(n, kv, -1, dim)
    starts, rows, before = s["starts"].long()[:-1], s["rows"].long(), s["lengths"].long() - s["rows"]
    token = (starts[:, None] + torch.arange(most, device="cuda")).clamp(max=s["tokens"] - 1)   # [n, most]
    # which keys: those before the step's, and of the step's rows the ancestors
    key = torch.arange(keys.shape[2], device="cuda")
    j = (key - before[:, None])[:, None, :]                                                # [n, 1, keys]
    word = s["masks"][token].gather(2, (j.clamp(0, most - 1) // 64).expand(n, most, -1))
    ancestor = (word >> (j.clamp(min=0) % 64)) & 1 > 0
    seen = (j < 0) | (ancestor & (j < rows[:, None, None]))
    if case["window"]:
        position = s["positions"].long()[token]
        of_key = torch.where(j[:, 0] < 0, key, position.gather(1, j[:, 0].clamp(0, most - 1)))
        seen &= of_key[:, None, :] > position[:, :, None] - case["window"]
    q = s["q"][:, token].permute(1, 0, 2, 3).reshape(n, kv, group * most, dim)
    scores = torch.matmul(q, keys.transpose(2, 3)) * (1.0 / math.sqrt(dim))
    scores = scores.view(n, kv, group, most, -1).masked_fill(~seen[:, None, None], -math.inf)
    weight = torch.exp(scores - scores.amax(-1, keepdim=True).clamp(min=-1e30))
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight.view(n, kv, group * most, -1), values).view(n, kv, group, most, dim) / total
    out = out.permute(0, 3, 1, 2, 4).reshape(n, most, heads * dim)
    index = torch.arange(s["tokens"], device="cuda") - starts[s["request"]]
    return out[s["request"], index]


def _plain_verify(s):
    """Row by row of all requests: a row whose parent is the last kept one is tried.  In 64 bits: a random number next to
    a border must fall to its side."""
    case, n, vocab = s["case"], s["case"]["requests"], s["case"]["vocab"]
    starts, rows = s["starts"].long()[:-1], s["rows"].long()
    every, warm = torch.arange(n, device="cuda"), s["temperatures"].double()[:, None]
    token_of = torch.arange(vocab, device="cuda")

    def first_largest(x):
        return torch.where(x == x.amax(1, keepdim=True), token_of, vocab).amin(1)

    def weights(logits, row):
        x = logits[starts + row].double()
        x = torch.exp((x - x.amax(1, keepdim=True)) / warm)
        return x, x.sum(1)

    current = torch.zeros_like(starts)
    used = torch.zeros(n, dtype=torch.float64, device="cuda")                              # C
    banned = torch.zeros(n, vocab, dtype=torch.bool, device="cuda")

    def left():
        """At the current rows: what is left of the target's weights, their sum, and the draft's probabilities in these units."""
        w, z = weights(s["logits"], current)
        if s["draft"] is None:
            r = w.masked_fill(banned, 0)
            return r, r.sum(1), None, w, z
        q, zq = weights(s["draft"], current)
        q *= (z / zq)[:, None]
        r = torch.where(used[:, None] > 0, (w - used[:, None] * q).clamp_(min=0), w)
        return r, r.sum(1), q, w, z

    kept = torch.ones_like(starts)
    path = torch.full((n, case["rows"]), -1, device="cuda")
    path[:, 0] = 0
    for i in range(1, s["max_rows"]):
        token = (starts + i).clamp(max=s["tokens"] - 1)
        tried = (i < rows) & (s["parents"].long()[token] == current)
        x = s["ids"].long()[token]
        if case["greedy"]:
            taken = tried & (first_largest(s["logits"][starts + current]) == x)
        else:
            r, total, q, _, z = left()
            u = s["accept"].double()[token]
            of_draft = u * total if q is None else u * total * q[every, x] / z
            taken = tried & (of_draft < r[every, x])
            refused = tried & ~taken
            used = torch.where(refused, used + total / z, torch.where(taken, 0, used))
            banned.masked_fill_(taken[:, None], False)
            banned[every, x] |= refused
        path[every, kept.clamp(max=case["rows"] - 1)] = torch.where(
            taken, i, path[every, kept.clamp(max=case["rows"] - 1)])
        kept = kept + taken
        current = torch.where(taken, i, current)
    if case["greedy"]:
        chosen = first_largest(s["logits"][starts + current])
    else:
        r, total, _, w, z = left()
        r = torch.where((total > 0)[:, None], r, w)
        chosen = (r.cumsum(1) <= (s["sample"].double() * r.sum(1))[:, None]).sum(1)
        chosen = torch.minimum(chosen, torch.where(r > 0, token_of, 0).amax(1))
    index = torch.arange(s["tokens"], device="cuda") - starts[s["request"]]
    return {"path": path[s["request"], index].int(), "kept": kept.int(), "next": chosen.int()}


def _plain_keep(s):
    case, block, n = s["case"], s["case"]["block"], s["case"]["requests"]
    starts, rows, kept, lengths = s["starts"].long()[:-1], s["rows"].long(), s["kept"].long(), s["lengths"].long()
    table, width = s["table"].long(), s["width"]
    before = lengths - rows
    # kept row k of a request: from place `path` to place k behind the cached tokens
    index = torch.arange(s["tokens"], device="cuda") - starts[s["request"]]
    moves = index < kept[s["request"]]

    def slot_of(place):
        position = (before[s["request"]] + place).clamp(min=0)
        return table[s["request"], position // block].clamp(min=0), position % block
    to, to_slot = slot_of(torch.where(moves, index, 0))
    source, source_slot = slot_of(torch.where(moves, s["path"].long(), 0))
    # the block that holds the last cached tokens keeps them
    last = table[torch.arange(n, device="cuda"), (before // block).clamp(max=width - 1)].clamp(min=0)
    shared = (before % block > 0) & (kept > 0)
    older = torch.zeros(s["blocks"], dtype=torch.long, device="cuda").scatter_reduce(
        0, last, torch.where(shared, before % block, 0), "amax")
    touched = torch.zeros(s["blocks"], dtype=torch.bool, device="cuda")
    touched = touched.long().scatter_reduce(0, to, moves.long(), "amax") > 0
    for codes, scales, transposed in ((s["keys"], s["key_scales"], False), (s["values"], s["value_scales"], True)):
        kv = case["kv_heads"]
        comes = torch.where(moves[:, None], scales[:, source], 0)                          # [layers, tokens, kv]
        new = torch.where((older > 0)[:, None], scales, 0).scatter_reduce(
            1, to[:, None].expand(-1, kv).expand_as(comes), comes, "amax")
        new = torch.where(touched[:, None], new, scales)
        view = codes.transpose(-1, -2) if transposed else codes                            # [layers, blocks, kv, block, dim]
        held = view.float().double()
        moved = held[:, source, :, source_slot] * (scales[:, source].double() / new[:, to].double())[..., None].permute(1, 0, 2, 3)
        stays = (torch.arange(block, device="cuda") < older[:, None]) & touched[:, None]
        ratio = (scales.double() / new.double())[..., None, None]
        held = torch.where(stays[None, :, None, :, None], held * ratio, held)
        held = held.permute(1, 3, 0, 2, 4)                                                 # [blocks, block, layers, kv, dim]
        at = torch.where(moves, to, s["blocks"])
        padded = torch.cat([held, held[:1]])
        padded[at, to_slot] = moved
        held = padded[:-1].permute(2, 0, 3, 1, 4)
        if case["form"] == INT8:
            held = held.round()
        view.copy_(held.float())
        scales.copy_(new)
    # blocks behind the kept tokens go on the free stack, in the requests' order
    after = before + kept
    first, end = (after + block - 1) // block, (lengths + block - 1) // block
    given, entry = end - first, torch.arange(width, device="cuda")
    at = s["count"].long() + (given.cumsum(0) - given)[:, None] + entry - first[:, None]
    at = torch.where((entry >= first[:, None]) & (entry < end[:, None]), at, s["blocks"])
    stack = torch.cat([s["stack"], s["stack"][:1]]).index_put((at,), s["table"])[:s["blocks"]]
    return _kept(s, after.int(), stack, (s["count"] + given.sum()).int())


# -------------------------------------------------------- work and accuracy ---
def work(case):
    cached, rows, parents = _plan(case)
    n, tokens = case["requests"], int(rows.sum())
    if case["kind"] == "tree":
        return {"bytes": 4 * tokens + 12 * n + tokens * (4 + 8 * _blocks_of(int(rows.max()), 64)), "flops": 0}
    if case["kind"] == "attend":
        heads, kv, dim, window = case["heads"], case["kv_heads"], case["dim"], case["window"] or 1 << 30
        keys, visible = 0, 0
        for c, f, tree in zip(cached.tolist(), rows.tolist(), parents):
            depth = _depths(tree)
            keys += min(c, window - 1) + f
            visible += int(np.minimum(c + depth + 1, window).sum())
        return {"bytes": 2 * kv * dim * keys + 8 * kv * _blocks_of(keys, case["block"]) + 8 * tokens * heads * dim
                + 8 * tokens * _blocks_of(int(rows.max()), 64), "flops": 4 * heads * dim * visible}
    if case["kind"] == "verify":
        # a walk reads the rows of one path: counted down to the tree's deepest row, which few walks reach
        read = sum(int(_depths(tree).max()) + 1 for tree in parents)
        ahead = sum(int(_depths(tree).max()) for tree in parents) if case["draft"] else 0
        return {"bytes": 4 * case["vocab"] * (read + ahead) + 16 * tokens + 16 * n,
                "flops": 0 if case["greedy"] else 4 * case["vocab"] * (read + ahead)}
    moved = sum(sum(k != j for k, j in enumerate(path)) for path in _paths(case))
    kept = np.array([len(path) for path in _paths(case)])
    block = case["block"]
    blocks = int((_blocks_of(cached + kept, block) - cached // block).sum())
    return {"bytes": case["layers"] * case["kv_heads"] * (4 * moved * case["dim"] + 16 * blocks) + 4 * tokens + 24 * n,
            "flops": 0}


def exact(case, seed):
    """In 64 bits; whole numbers have no such value."""
    if case["kind"] in ("tree", "verify"):
        return None
    s = prepare(case, seed)
    cached, rows, parents = _plan(case)
    starts = np.concatenate([[0], np.cumsum(rows)])
    block, form = case["block"], case["form"]
    if case["kind"] == "attend":
        heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
        group = heads // kv
        out = torch.empty(s["tokens"], heads, dim, dtype=torch.float64, device="cuda")
        for r, (c, f, tree) in enumerate(zip(cached.tolist(), rows.tolist(), parents)):
            depth = _depths(tree)
            where = np.concatenate([np.arange(c), c + depth])                              # positions of the keys
            seen = np.concatenate([np.ones((f, c), bool), _ancestors(tree)], 1)
            if case["window"]:
                seen &= where[None, :] > (c + depth)[:, None] - case["window"]
            hidden = torch.as_tensor(~seen, device="cuda")
            pages = s["table"][r, :_blocks_of(c + f, block)].long()
            for h in range(kv):
                k = s["keys"][pages, h].double() * s["key_scales"][pages, h].double()[:, None, None]
                v = s["values"][pages, h].double() * s["value_scales"][pages, h].double()[:, None, None]
                k, v = k.reshape(-1, dim)[:c + f], v.transpose(1, 2).reshape(-1, dim)[:c + f]
                q = s["q"][h * group:(h + 1) * group, starts[r]:starts[r] + f].double()
                for g in range(group):
                    score = (q[g] @ k.T / math.sqrt(dim)).masked_fill(hidden, -math.inf)
                    out[starts[r]:starts[r] + f, h * group + g] = torch.softmax(score, -1) @ v
        return out.reshape(s["tokens"], heads * dim)
    table, result = s["table"].cpu().numpy(), {}
    for name in ("keys", "values"):
        scales = s[name[:-1] + "_scales"].cpu().numpy().astype(np.float64)                 # [layers, blocks, kv]
        held = s[name].cpu().float().numpy().astype(np.float64)
        held = held.transpose(0, 1, 2, 4, 3).copy() if name == "values" else held          # [layers, blocks, kv, block, dim]
        was, scale_was = held.copy(), scales.copy()
        for r, path in enumerate(_paths(case)):
            page = table[r]
            comes = {}                                   # of a block: (its slot, where that token comes from)
            for position in range(int(cached[r]) // block * block, int(cached[r]) + len(path)):
                place = position - int(cached[r])
                origin = position if place < 0 else int(cached[r]) + path[place]
                comes.setdefault(page[position // block], []).append(
                    (position % block, page[origin // block], origin % block, place))
            for to, tokens in comes.items():
                if all(place < 0 for _, _, _, place in tokens):
                    continue
                scale = np.max([scale_was[:, source] for _, source, _, _ in tokens], 0)    # [layers, kv]
                for slot, source, source_slot, _ in tokens:
                    ratio = (scale_was[:, source] / scale)[..., None]
                    held[:, to, :, slot] = _nearest(was[:, source, :, source_slot] * ratio, form)
                scales[:, to] = scale
        stood = held * scales[..., None, None]
        stood = stood.transpose(0, 1, 2, 4, 3).copy() if name == "values" else stood
        result[name], result[name[:-1] + "_scales"] = torch.from_numpy(stood), torch.from_numpy(scales)
    order = ("keys", "values", "key_scales", "value_scales")
    return {**{k: result[k] for k in order}, "lengths": None, "stack": None, "left": None}


def _nearest(x, form):
    """The nearest code, ties to even: a whole number, or a value of three mantissa bits down to 2^-9."""
    if form == INT8:
        return np.clip(np.rint(x), -127, 127)
    step = np.exp2(np.maximum(np.floor(np.log2(np.maximum(np.abs(x), 2.0 ** -20))), -6) - 3)
    return np.rint(x / step) * step

"""The operators of the 8-bit KV cache in blocks: what is timed, and their plain forms.

A program that serves several requests keeps their keys and values in one pool
of blocks, 8 bits a value with a scale for each block and KV head:

* ``assign``: a step's block tables and slot maps, from the requests' lengths;
* ``append``: RoPE, and the step's keys and values quantized into their blocks;
* ``attend``: causal grouped-query attention of the step's tokens over the blocks.

Head layouts are those of the presets in ``leaf_amd/models.py`` and of the
tests; lengths run from single tokens behind a few keys to whole prompts.
``run`` computes them from elementary torch operations, or with ``own`` calls
the library.
"""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import torch

own = False

# (heads, kv_heads, dim): the presets' layouts, heads of 128 and of 80, and the reduced presets' width.
LAYOUTS = ((32, 4, 64), (14, 2, 64), (15, 5, 64), (12, 12, 64), (32, 8, 128), (8, 2, 80), (8, 2, 32))
INT8, E4M3 = 0, 1
SMALLEST = {INT8: 1e-12, E4M3: 2.0 ** -40}


# ------------------------------------------------------------------- cases ---
def _assign(requests, fresh, longest, block, ended=0, mix=1):
    return {"kind": "assign", "requests": requests, "fresh": fresh, "longest": longest, "block": block,
            "ended": ended, "mix": mix}


def _append(requests, chunks, rows, layout, block, form, mix=1):
    heads, kv_heads, dim = layout
    return {"kind": "append", "requests": requests, "chunks": chunks, "rows": rows, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "block": block, "form": form, "shortest": 0, "longest": block - 1,
            "mix": mix}


def _attend(requests, chunks, rows, shortest, longest, layout, block, form, window=0, mix=1):
    heads, kv_heads, dim = layout
    return {"kind": "attend", "requests": requests, "chunks": chunks, "rows": rows, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "block": block, "form": form, "shortest": shortest,
            "longest": longest, "window": window, "mix": mix}


def listed():
    cases = {
        # A decode step of a small server: one token for each of 24 requests, the smallest call.
        "assign_decode": _assign(24, 1, 2000, 16),
        # A step that takes in a burst of ragged prompts.
        "assign_prompts": _assign(40, 777, 0, 64),
        # A large server's decode step in which one request in twenty has ended.
        "assign_churn": _assign(1000, 1, 4000, 16, ended=50),
        # A decode step's keys and values, heads grouped by eight.
        "append_decode": _append(64, 0, 1, (32, 4, 64), 16, INT8),
        # A whole prompt of 2048 tokens.
        "append_prompt": _append(1, 1, 2048, (14, 2, 64), 64, INT8),
        # A prompt's chunk beside 47 requests that decode, 8-bit floating point, heads of 128.
        "append_mixed": _append(48, 1, 500, (32, 8, 128), 32, E4M3),
        # One request decodes at a context of 4095 tokens.
        "attend_single": _attend(1, 0, 1, 4095, 4095, (14, 2, 64), 64, INT8),
        # 64 requests decode at ragged contexts, heads of 128 grouped by four.
        "attend_batch": _attend(64, 0, 1, 200, 4096, (32, 8, 128), 64, INT8),
        # 100 short conversations in small blocks of 8-bit floating point, heads grouped by three.
        "attend_batch_e4m3": _attend(100, 0, 1, 30, 2000, (15, 5, 64), 16, E4M3),
        # A prompt of 2048 tokens from its first.
        "attend_prompt": _attend(1, 1, 2048, 0, 0, (14, 2, 64), 64, INT8),
        # A chunk of 512 tokens behind a long cached context.
        "attend_chunk": _attend(1, 1, 512, 7001, 7001, (32, 8, 128), 32, E4M3),
        # A prompt's chunk beside 24 requests that decode, sliding window.
        "attend_mixed": _attend(25, 1, 384, 300, 3000, (32, 4, 64), 32, INT8, window=1024),
    }
    return [dict(case, name=name) for name, case in cases.items()]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("assign", "append", "attend", "attend"))
    block, mix = rng.choice((16, 32, 64, 128)), rng.randint(2, 1 << 20)
    if kind == "assign":
        requests = _log_int(rng, 1, 2000)
        fresh = rng.choice((1, 1, min(1000, max(2, 30000 // requests))))
        ended = requests // 20 if rng.random() < 0.5 else 0
        return _assign(requests, fresh, _log_int(rng, 100, 8000), block, ended, mix)
    layout, form = rng.choice(LAYOUTS), rng.choice((INT8, E4M3))
    heads, kv_heads, dim = layout
    if kind == "append":
        requests = _log_int(rng, 1, 200)
        chunks = rng.choice((0, 1, min(requests, 3)))
        return _append(requests, chunks, _log_int(rng, 2, 1500) if chunks else 1, layout, block, form, mix)
    shape = rng.choice(("decode", "decode", "prompt", "chunk", "mixed"))
    window = rng.choice((0, 0, 0, 512))
    if shape == "decode":
        longest = _log_int(rng, 20, 16000)
        requests = min(_log_int(rng, 1, 200), max(1, int(2.5e8 / (kv_heads * dim * longest))))
        return _attend(requests, 0, 1, max(1, longest // 20), longest, layout, block, form, window, mix)
    if shape == "prompt":
        return _attend(1, 1, _log_int(rng, 2, 2048), 0, 0, layout, block, form, window, mix)
    if shape == "chunk":
        rows, longest = _log_int(rng, 2, 512), _log_int(rng, 16, 7000)
        return _attend(1, 1, rows, longest, longest, layout, block, form, window, mix)
    rows, longest = _log_int(rng, 2, 400), _log_int(rng, 50, 3000)
    requests = min(rng.randint(2, 40), max(2, int(6e8 / (heads * rows * (longest + rows)))))
    return _attend(requests, 1, rows, longest // 10, longest, layout, block, form, window, mix)


def _requests(case):
    """(cached, fresh) of each request: ragged, the same for every seed, so that the work is."""
    r, n = np.random.RandomState(case["mix"]), case["requests"]
    if case["kind"] == "assign":
        cached = r.randint(0, case["longest"] + 1, n)
        fresh = r.randint(1, case["fresh"] + 1, n)
        fresh[r.permutation(n)[:case["ended"]]] = -1
        return cached, fresh
    cached = r.randint(case["shortest"], case["longest"] + 1, n)
    fresh = np.ones(n, int)
    where = r.permutation(n)[:case["chunks"]]
    fresh[where] = case["rows"]
    return cached, fresh


def _blocks_of(tokens, block):
    return -(-tokens // block)


# ------------------------------------------------------------------ inputs ---
def _ints(a):
    return torch.as_tensor(np.ascontiguousarray(a), dtype=torch.int32, device="cuda")


def _codes(gen, count, shape, form):
    """Codes of N(0, 1) values under scales that differ from block to block."""
    x = torch.randn(shape, generator=gen, device="cuda")
    scale = torch.exp(0.3 * torch.randn(count, generator=gen, device="cuda")) * (4.0 / 127 if form == INT8 else 2.0 ** -6)
    if form == INT8:
        return (32 * x).round_().clamp_(-127, 127).to(torch.int8), scale
    return (64 * x).clamp_(-448, 448).to(torch.float8_e4m3fn), torch.exp2(torch.round(torch.log2(scale)))


def _rope_tables(positions, dim):
    angle = np.arange(positions, dtype=np.float32)[:, None] * \
        (np.float32(10000.0) ** (-np.arange(0, dim, 2, dtype=np.float32) / np.float32(dim)))[None, :]
    return torch.from_numpy(np.cos(angle)).cuda().contiguous(), torch.from_numpy(np.sin(angle)).cuda().contiguous()


def _prepare_assign(case, gen, s):
    cached, fresh = _requests(case)
    block, n = case["block"], case["requests"]
    held = _blocks_of(cached, block)
    width = int(_blocks_of(cached + np.maximum(fresh, 0), block).max())
    needed = int((_blocks_of(cached + np.maximum(fresh, 0), block) - held).sum())
    # a pool that just suffices for most of the step: the last requests may be turned away
    blocks = int(held.sum()) + needed - needed // 50
    order = torch.randperm(blocks, generator=gen, device="cuda").int()
    entry = torch.arange(width, device="cuda")
    first = _ints(np.cumsum(held) - held)
    table = torch.where(entry < _ints(held)[:, None], order[(first[:, None] + entry).clamp(max=blocks - 1)], -1)
    stack = torch.full((blocks,), -1, dtype=torch.int32, device="cuda")
    stack[:blocks - int(held.sum())] = order[int(held.sum()):]
    tokens = int(np.maximum(fresh, 0).sum())
    return dict(s, cached=_ints(cached), fresh=_ints(fresh), table=table.int().contiguous(), stack=stack,
                count=_ints([blocks - int(held.sum())]), left=_ints([0]), starts=_ints(np.zeros(n + 1)),
                rows=_ints(np.zeros(n)), lengths=_ints(np.zeros(n)), positions=_ints(np.zeros(tokens)),
                slots=_ints(np.zeros(tokens)), blocks=blocks, width=width, tokens=tokens, max_rows=case["fresh"])


def _prepare_batch(case, gen, s):
    """A step's plan as an earlier call has left it, over a pool that holds the blocks of all requests."""
    cached, fresh = _requests(case)
    block, n = case["block"], case["requests"]
    # (an append reaches no block but a request's last and new ones: its cases hold no others)
    lengths, starts = cached + fresh, np.concatenate([[0], np.cumsum(fresh)])
    held = _blocks_of(lengths, block)
    blocks, width, tokens = int(held.sum()), int(held.max()), int(fresh.sum())
    order = torch.randperm(blocks, generator=gen, device="cuda").int()
    entry = torch.arange(width, device="cuda")
    first = _ints(np.cumsum(held) - held)
    table = torch.where(entry < _ints(held)[:, None], order[(first[:, None] + entry).clamp(max=blocks - 1)], -1)
    request = np.repeat(np.arange(n), fresh)
    position = cached[request] + np.arange(tokens) - starts[request]
    slots = table.long()[torch.as_tensor(request, device="cuda"), torch.as_tensor(position // block, device="cuda")] * block \
        + torch.as_tensor(position % block, device="cuda")
    kv, dim = case["kv_heads"], case["dim"]
    keys, key_scales = _codes(gen, blocks * kv, (blocks, kv, block, dim), case["form"])
    values, value_scales = _codes(gen, blocks * kv, (blocks, kv, dim, block), case["form"])
    return dict(s, lengths=_ints(lengths), rows=_ints(fresh), starts=_ints(starts), table=table.int().contiguous(),
                positions=_ints(position), slots=slots.int(), request=torch.as_tensor(request, device="cuda"),
                keys=keys, values=values, key_scales=key_scales.view(blocks, kv), value_scales=value_scales.view(blocks, kv),
                blocks=blocks, width=width, tokens=tokens, max_rows=int(fresh.max()))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    if case["kind"] == "assign":
        s = _prepare_assign(case, gen, s)
    else:
        s = _prepare_batch(case, gen, s)
        heads, kv, dim, tokens = case["heads"], case["kv_heads"], case["dim"], s["tokens"]
        if case["kind"] == "append":
            s["qkv"] = torch.randn(tokens, (heads + 2 * kv) * dim, generator=gen, device="cuda")
            s["cos"], s["sin"] = _rope_tables(int(s["positions"].max()) + 1, dim)
            s["q"] = torch.empty(heads, tokens, dim, device="cuda")
        else:
            s["q"] = torch.randn(heads, tokens, dim, generator=gen, device="cuda")
            s["out"] = torch.empty(tokens, heads * dim, device="cuda")
    if own:
        _describe(s)
    return s


def _describe(s):
    """The library's descriptions of the batch and the cache, which a program keeps from step to step."""
    from leaf_amd import runtime
    case = s["case"]

    def at(name):
        return s[name].data_ptr() if name in s else None
    s["batch"] = runtime.KvBatch(
        requests=case["requests"], tokens=s["tokens"], max_rows=s["max_rows"], block=case["block"], blocks=s["blocks"],
        width=s["width"], cached=at("cached"), fresh=at("fresh"), free_blocks=at("stack"), free_count=at("count"),
        free_left=at("left"), table=at("table"), lengths=at("lengths"), starts=at("starts"), rows=at("rows"),
        positions=at("positions"), slots=at("slots"))
    if case["kind"] != "assign":
        s["cache"] = runtime.Kv8(keys=at("keys"), values=at("values"), key_scales=at("key_scales"),
                                 value_scales=at("value_scales"), kv_heads=case["kv_heads"], dim=case["dim"],
                                 format=case["form"])
    s["lib"], s["check"] = runtime.library(), runtime.check


# -------------------------------------------------------------------- runs ---
def run(state):
    kind = state["case"]["kind"]
    if kind == "assign":
        return _own_assign(state) if own else _plain_assign(state)
    if kind == "append":
        return _own_append(state) if own else _plain_append(state)
    return _own_attend(state) if own else _plain_attend(state)


def _own_assign(s):
    s["check"](s["lib"].lh_kv_assign(C.byref(s["batch"]), None))
    return {key: s[key] for key in ("table", "stack", "left", "starts", "rows", "lengths", "positions", "slots")}


def _own_append(s):
    case = s["case"]
    s["check"](s["lib"].lh_rope_kv8(C.byref(s["batch"]), C.byref(s["cache"]), s["qkv"].data_ptr(), case["heads"],
                                    case["dim"], s["cos"].data_ptr(), s["sin"].data_ptr(), s["cos"].shape[0],
                                    s["q"].data_ptr(), None))
    return _appended(s)


def _own_attend(s):
    case = s["case"]
    s["check"](s["lib"].lh_attention_kv8(C.byref(s["batch"]), C.byref(s["cache"]), s["q"].data_ptr(), case["heads"],
                                         case["window"], s["out"].data_ptr(), None, 0, None))
    return s["out"]


def _values_of(codes, scales):
    """What codes stand for."""
    if codes.dtype == torch.int8:
        return codes * scales[:, :, None, None]
    return codes.float().mul_(scales[:, :, None, None])


def _appended(s):
    return {"q": s["q"], "keys": _values_of(s["keys"], s["key_scales"]),
            "values": _values_of(s["values"], s["value_scales"]), "key_scales": s["key_scales"],
            "value_scales": s["value_scales"]}


def _plain_assign(s):
    case, block, width, blocks = s["case"], s["case"]["block"], s["width"], s["blocks"]
    cached, fresh, count = s["cached"].long(), s["fresh"].long(), s["count"].long()
    entry = torch.arange(width, device="cuda")
    ended, new = fresh < 0, fresh.clamp(min=0)
    held = (cached + block - 1) // block
    # blocks of ended requests go on the free stack, in the requests' order
    given = torch.where(ended, held, 0)
    at = count + (given.cumsum(0) - given)[:, None] + entry
    at = torch.where(entry < given[:, None], at, blocks)
    stack = torch.cat([s["stack"], s["stack"][:1]]).index_put((at,), s["table"])[:blocks]
    free = count + given.sum()
    # new blocks from the top of the stack, as long as it lasts
    starts = torch.cat([torch.zeros_like(new[:1]), new.cumsum(0)])
    after = cached + new
    fits = ~ended & (after <= width * block) & (new <= s["max_rows"]) & (starts[1:] <= s["tokens"])
    need = torch.where(fits, (after + block - 1) // block - held, 0)
    upto = need.cumsum(0)
    takes = fits & ((need == 0) | (upto <= free))
    need = torch.where(takes, need, 0)
    place = entry - held[:, None]
    fill = (place >= 0) & (place < need[:, None])
    taken = stack[(free - 1 - ((upto - need)[:, None] + place)).clamp(0, blocks - 1)]
    table = torch.where(fill, taken, s["table"])
    rows = torch.where(takes, new, 0)
    # a position and a slot for each token
    token = torch.arange(s["tokens"], device="cuda")
    request = torch.searchsorted(starts[1:].contiguous(), token, right=True).clamp(max=case["requests"] - 1)
    position = cached[request] + token - starts[request]
    valid = takes[request] & (token < starts[-1])
    slot = table[request, (position // block).clamp(0, width - 1)].long() * block + position % block
    return {"table": table, "stack": stack, "left": (free - need.sum()).int(), "starts": starts.int(), "rows": rows.int(),
            "lengths": torch.where(ended, 0, cached + rows).int(),
            "positions": torch.where(valid, position, -1).int(), "slots": torch.where(valid, slot, -1).int()}


def _quantized(codes, scales, x, slots, block, form, transposed):
    """The run's rows x [tokens, kv_heads, dim] into their blocks, whose older codes follow a scale that grew."""
    kv, dim = x.shape[1:]
    at, offset = slots // block, slots % block
    biggest = x.abs().amax(-1)
    first = torch.full((len(codes),), block, device="cuda").scatter_reduce(0, at, offset, "amin")
    touched = first < block
    amax = torch.zeros_like(scales).scatter_reduce(0, at[:, None].expand(-1, kv), biggest, "amax")
    if form == INT8:
        need = (amax.double() / 127).float().clamp_min(SMALLEST[form])
    else:
        mantissa, exponent = torch.frexp(amax)          # mantissa in [0.5, 1): 448 = 0.875 * 2^9
        need = torch.ldexp(torch.ones_like(amax), exponent - 9 + (mantissa > 0.875).int()).clamp_min(SMALLEST[form])
    before = torch.where((first > 0)[:, None] & touched[:, None], scales, 0)
    scale = torch.where(touched[:, None], torch.maximum(before, need), scales)
    grown = (touched & (first > 0))[:, None] & (scale > before)
    older = torch.arange(block, device="cuda") < first[:, None]
    older = (older[:, None, None, :] if transposed else older[:, None, :, None]) & grown[:, :, None, None]
    moved = codes.double()
    moved = torch.where(older, moved * before.double()[:, :, None, None] / scale.double()[:, :, None, None], moved)
    fresh = x.double() / scale[at].double()[:, :, None]
    if form == INT8:
        moved, fresh = moved.round(), fresh.round().clamp(-127, 127)
    target = moved.permute(0, 3, 1, 2) if transposed else moved.permute(0, 2, 1, 3)      # [blocks, block, kv, dim]
    target.index_put_((at, offset), fresh)
    codes.copy_(moved.float())
    scales.copy_(scale)


def _plain_append(s):
    case = s["case"]
    heads, kv, dim, block = case["heads"], case["kv_heads"], case["dim"], case["block"]
    rows = s["qkv"].view(-1, heads + 2 * kv, dim)
    c, sn = s["cos"][s["positions"].long()][:, None], s["sin"][s["positions"].long()][:, None]
    a, b = rows[:, :heads + kv, :dim // 2], rows[:, :heads + kv, dim // 2:]
    turned = torch.cat([a * c - b * sn, b * c + a * sn], -1)
    s["q"].copy_(turned[:, :heads].transpose(0, 1))
    slots = s["slots"].long()
    _quantized(s["keys"], s["key_scales"], turned[:, heads:], slots, block, case["form"], False)
    _quantized(s["values"], s["value_scales"], rows[:, heads + kv:], slots, block, case["form"], True)
    return _appended(s)


def _plain_attend(s):
    case = s["case"]
    heads, kv, dim, n, most = case["heads"], case["kv_heads"], case["dim"], case["requests"], s["max_rows"]
    group = heads // kv
    table = s["table"].long().clamp(min=0)
    keys = s["keys"].float()[table] * s["key_scales"][table][..., None, None]              # [n, width, kv, block, dim]
    values = s["values"].float()[table] * s["value_scales"][table][..., None, None]        # [n, width, kv, dim, block]
    keys = keys.permute(0, 2, 1, 3, 4).reshape(n, kv, -1, dim)
    values = values.permute(0, 2, 1, 4, 3).reshape(n, kv, -1, dim)
    starts, rows, lengths = s["starts"].long()[:-1], s["rows"].long(), s["lengths"].long()
    row = torch.arange(most, device="cuda")
    token = (starts[:, None] + row).clamp(max=s["tokens"] - 1)                             # [n, most]
    q = s["q"][:, token].permute(1, 0, 2, 3).reshape(n, kv, group * most, dim)
    scores = torch.matmul(q, keys.transpose(2, 3)) * (1.0 / math.sqrt(dim))
    key, query = torch.arange(keys.shape[2], device="cuda"), ((lengths - rows)[:, None] + row)[:, :, None]
    seen = (key <= query) & (key < lengths[:, None, None])
    if case["window"]:
        seen &= key > query - case["window"]
    scores = scores.view(n, kv, group, most, -1).masked_fill(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-1e30)
    weight = torch.exp(scores - top)
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight.view(n, kv, group * most, -1), values).view(n, kv, group, most, dim) / total
    out = out.permute(0, 3, 1, 2, 4).reshape(n, most, heads * dim)
    index = torch.arange(s["tokens"], device="cuda") - starts[s["request"]]
    return out[s["request"], index]


# -------------------------------------------------------- work and accuracy ---
def work(case):
    cached, fresh = _requests(case)
    block, n = case["block"], case["requests"]
    if case["kind"] == "assign":
        new = np.maximum(fresh, 0)
        tokens, needed = int(new.sum()), int((_blocks_of(cached + new, block) - _blocks_of(cached, block)).sum())
        given = int(_blocks_of(cached, block)[fresh < 0].sum())
        return {"bytes": 4 * (2 * n + 3 * n + 1 + 2 * tokens + 2 * needed + 2 * given + 2), "flops": 0}
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    tokens = int(fresh.sum())
    if case["kind"] == "append":
        runs = int((_blocks_of(cached + fresh, block) - cached // block).sum())
        return {"bytes": 4 * tokens * (2 * heads + 2 * kv) * dim + 2 * tokens * kv * dim + 8 * tokens
                + 4 * dim * min(tokens, block + case["rows"]) + 16 * runs * kv,
                "flops": 6 * tokens * (heads + kv) * dim // 2 + 4 * tokens * kv * dim}
    window = case["window"] or 1 << 30
    keys, visible = 0, 0
    for c, f in zip(cached.tolist(), fresh.tolist()):
        keys += min(c + f, window + f - 1)
        seen = np.minimum(np.arange(c + 1, c + f + 1), window)
        visible += int(seen.sum())
    return {"bytes": 2 * kv * dim * keys + 8 * kv * _blocks_of(keys, block) + 8 * tokens * heads * dim,
            "flops": 4 * heads * dim * visible}


def exact(case, seed):
    """In 64 bits.  A cached key is quantized from the f32 row that RoPE is defined to give (each product and their
    difference rounded); the query is what the rotation is in 64 bits."""
    if case["kind"] == "assign":
        return None
    s = prepare(case, seed)
    heads, kv, dim, block, form = case["heads"], case["kv_heads"], case["dim"], case["block"], case["form"]
    group = heads // kv
    if case["kind"] == "attend":
        out = torch.empty(s["tokens"], heads, dim, dtype=torch.float64, device="cuda")
        for r, (first, count, length) in enumerate(zip(s["starts"].tolist(), s["rows"].tolist(), s["lengths"].tolist())):
            pages = s["table"][r, :_blocks_of(length, block)].long()
            p = torch.arange(length - count, length, device="cuda")[:, None]
            j = torch.arange(length, device="cuda")[None]
            hidden = (j > p) | ((j <= p - case["window"]) if case["window"] else (j < 0))
            for h in range(kv):
                k = s["keys"][pages, h].double() * s["key_scales"][pages, h].double()[:, None, None]
                v = s["values"][pages, h].double() * s["value_scales"][pages, h].double()[:, None, None]
                k, v = k.reshape(-1, dim)[:length], v.transpose(1, 2).reshape(-1, dim)[:length]
                q = s["q"][h * group:(h + 1) * group, first:first + count].double()
                score = torch.stack([(one @ k.T / math.sqrt(dim)).masked_fill(hidden, -math.inf) for one in q])
                out[first:first + count, h * group:(h + 1) * group] = (torch.softmax(score, -1) @ v).transpose(0, 1)
        return out.reshape(s["tokens"], heads * dim)
    rows = s["qkv"].cpu().numpy().reshape(-1, heads + 2 * kv, dim)
    positions, slots = s["positions"].cpu().numpy(), s["slots"].cpu().numpy()
    c, sn = s["cos"].cpu().numpy()[positions][:, None], s["sin"].cpu().numpy()[positions][:, None]
    half = dim // 2
    low, high = rows[:, :heads, :half].astype(np.float64), rows[:, :heads, half:].astype(np.float64)
    q = np.concatenate([low * c - high * sn, high * c + low * sn], -1).transpose(1, 0, 2)
    low, high = rows[:, heads:heads + kv, :half], rows[:, heads:heads + kv, half:]
    fresh = {"keys": np.concatenate([low * c - high * sn, high * c + low * sn], -1), "values": rows[:, heads + kv:]}
    out = {"q": torch.from_numpy(q)}
    begins = [0] + [t for t in range(1, len(slots)) if slots[t] != slots[t - 1] + 1 or slots[t] % block == 0] + [len(slots)]
    for name in ("keys", "values"):
        scales = s[name[:-1] + "_scales"].cpu().numpy().astype(np.float64)
        held = s[name].cpu().float().numpy().astype(np.float64)
        held = np.ascontiguousarray(held.transpose(0, 1, 3, 2) if name == "values" else held)
        for a, b in zip(begins, begins[1:]):
            page, first = divmod(int(slots[a]), block)
            run = fresh[name][a:b].astype(np.float64).transpose(1, 0, 2)                   # [kv, tokens, dim]
            most = np.abs(run).max((1, 2))
            if form == INT8:
                need = np.maximum((most / 127).astype(np.float32), np.float32(1e-12)).astype(np.float64)
            else:
                need = np.maximum(2.0 ** np.ceil(np.log2(most / 448)), 2.0 ** -40)
            old = scales[page] if first else np.zeros(kv)
            new = np.maximum(old, need)
            older = held[page, :, :first]
            moved = _nearest(older * old[:, None, None] / new[:, None, None], form)
            held[page, :, :first] = np.where((new > old)[:, None, None], moved, older)
            held[page, :, first:first + b - a] = _nearest(run / new[:, None, None], form)
            scales[page] = new
        stood = held * scales[:, :, None, None]
        out[name] = torch.from_numpy(np.ascontiguousarray(stood.transpose(0, 1, 3, 2) if name == "values" else stood))
        out[name[:-1] + "_scales"] = torch.from_numpy(scales)
    return out


def _nearest(x, form):
    """The nearest code, ties to even: a whole number, or a value of three mantissa bits down to 2^-9."""
    if form == INT8:
        return np.clip(np.rint(x), -127, 127)
    step = np.exp2(np.maximum(np.floor(np.log2(np.maximum(np.abs(x), 2.0 ** -20))), -6) - 3)
    return np.rint(x / step) * step

"""Plain 64-bit forms of the operators over an 8-bit KV cache in blocks (include/leafhip.h)."""
from __future__ import annotations

import numpy as np

INT8, E4M3 = 0, 1


def e4m3_values():
    """What the 256 codes stand for (0x7F and 0xFF: NaN)."""
    c = np.arange(256)
    exponent, mantissa = (c >> 3) & 15, c & 7
    v = np.where(exponent == 0, mantissa * 2.0 ** -9, (8 + mantissa) * 2.0 ** (exponent - 10.0))
    v[(c & 127) == 127] = np.nan
    return np.where(c & 128, -v, v)


E4M3_VALUES = e4m3_values()


def decode(codes, form):
    return codes.view(np.int8).astype(np.float64) if form == INT8 else E4M3_VALUES[codes]


def encode(x, form):
    """The nearest code of each value, ties to even."""
    if form == INT8:
        return np.clip(np.rint(x), -127, 127).astype(np.int8).view(np.uint8)
    size = np.abs(x)
    step = 2.0 ** (np.maximum(np.floor(np.log2(np.maximum(size, 2.0 ** -20))), -6) - 3)
    size = np.rint(size / step) * step
    positive = E4M3_VALUES[:127]
    return (np.searchsorted(positive, size) | np.where(np.signbit(x), 128, 0)).astype(np.uint8)


def needed_scale(most, form):
    if form == INT8:
        return max(np.float32(np.float64(most) / 127), np.float32(1e-12))
    scale = 2.0 ** -40
    while 448 * scale < most:
        scale *= 2
    return np.float32(scale)


def rotated(rows, cosines, sines):
    """rows [..., dim] in f32, each product and their difference rounded; cosines, sines [..., rotary / 2]."""
    half = cosines.shape[-1]
    out, a, b = rows.copy(), rows[..., :half], rows[..., half:2 * half]
    out[..., :half], out[..., half:2 * half] = a * cosines - b * sines, b * cosines + a * sines
    return out


def append(codes, scales, x, slots, block, form, transposed):
    """Rows x [tokens, kv_heads, dim] into codes and scales, in place; slots below 0 are skipped."""
    begins = [t for t in range(len(slots)) if slots[t] >= 0 and
              (t == 0 or slots[t] % block == 0 or slots[t] != slots[t - 1] + 1)]
    for t in begins:
        n = 1
        while t + n < len(slots) and slots[t + n] == slots[t] + n and slots[t + n] % block:
            n += 1
        page, offset = divmod(int(slots[t]), block)
        for h in range(x.shape[1]):
            held = codes[page, h].T if transposed else codes[page, h]
            run, old = x[t:t + n, h].astype(np.float64), scales[page, h] if offset else np.float32(0)
            held[offset:offset + n] = 0
            if not np.isfinite(run).all() or not np.isfinite(old):
                scales[page, h] = np.nan
                continue
            scale = max(needed_scale(np.abs(run).max(), form), old)
            if offset and scale > old:
                held[:offset] = encode(decode(held[:offset], form) * np.float64(old) / np.float64(scale), form)
            held[offset:offset + n] = encode(run / np.float64(scale), form)
            scales[page, h] = scale


def attention(q, keys, values, key_scales, value_scales, table, lengths, starts, rows, block, form, window, out):
    """q [heads, tokens, dim]; fills out [tokens, heads, dim] (f64) and returns the sum of |q||k| of the largest score."""
    heads, _, dim = q.shape
    group, largest = heads // keys.shape[1], 0.0
    blocks = len(keys)
    for r in range(len(rows)):
        if rows[r] <= 0 or lengths[r] < rows[r]:
            continue
        pages = table[r, :-(-lengths[r] // block)]
        known = (pages >= 0) & (pages < blocks)
        at = np.where(known, pages, 0)
        for kvh in range(keys.shape[1]):
            ks = np.where(known, key_scales[at, kvh], np.nan).astype(np.float64)
            vs = np.where(known, value_scales[at, kvh], np.nan).astype(np.float64)
            k = (decode(keys[at, kvh], form) * ks[:, None, None]).reshape(-1, dim)
            v = (decode(values[at, kvh], form) * vs[:, None, None]).transpose(0, 2, 1).reshape(-1, dim)
            for i in range(rows[r]):
                last = lengths[r] - rows[r] + i
                first = max(0, last + 1 - window) if window else 0
                for h in range(kvh * group, (kvh + 1) * group):
                    x = q[h, starts[r] + i].astype(np.float64)
                    s = k[first:last + 1] @ x / np.sqrt(dim)
                    if not np.isfinite(s).all() or not np.isfinite(v[first:last + 1]).all():
                        out[starts[r] + i, h] = np.nan
                        continue
                    p = np.exp(s - s.max())
                    out[starts[r] + i, h] = (p / p.sum()) @ v[first:last + 1]
                    largest = max(largest, float((np.abs(k[first:last + 1]) @ np.abs(x)).max()) / np.sqrt(dim))
    return largest


def assign(cached, fresh, table, stack, count, block, width, blocks, tokens, max_rows):
    """A step's plan, request by request: a dict of what lh_kv_assign writes."""
    cached, fresh = np.asarray(cached), np.asarray(fresh)
    n = len(cached)
    table, stack = table.copy(), stack.copy()
    held = [-(-int(c) // block) for c in cached]
    for r in range(n):
        if fresh[r] < 0:
            for j in range(held[r]):
                stack[count], count = table[r, j], count + 1
    stack_after = stack.copy()
    starts, rows, lengths = np.zeros(n + 1, int), np.zeros(n, int), np.zeros(n, int)
    positions, slots = np.full(tokens, -1), np.full(tokens, -1)
    wanted, used = 0, 0
    for r in range(n):
        new = max(int(fresh[r]), 0)
        starts[r + 1] = starts[r] + new
        lengths[r] = 0 if fresh[r] < 0 else cached[r]
        after = int(cached[r]) + new
        if fresh[r] < 0 or after > width * block or new > max_rows or starts[r + 1] > tokens:
            continue
        need = -(-after // block) - held[r]
        wanted += need
        if need and wanted > count:
            continue
        for j in range(need):
            table[r, held[r] + j] = stack[count - 1 - used - j]
        used += need
        rows[r], lengths[r] = new, after
        for i in range(new):
            p = int(cached[r]) + i
            positions[starts[r] + i], slots[starts[r] + i] = p, table[r, p // block] * block + p % block
    return {"table": table, "free_blocks": stack_after, "free_left": np.array([count - used]),
            "starts": np.minimum(starts, tokens), "rows": rows, "lengths": lengths, "positions": positions, "slots": slots}

"""The paged cache's operators from their definitions, in 64 bits, on the CPU.

Arguments are NumPy arrays (float64 values of what the GPU holds in fewer
bits); every function is a plain loop over requests, tokens and heads.
"""

import numpy as np


def paged_tables(past, fresh, table, free_pages, page_size, num_tokens):
    """(table, starts, requests, lengths, slots, used) as the library's
    paged_tables gives them; the table is a copy."""
    table = np.array(table, np.int64)
    width = table.shape[1]
    starts = np.concatenate([[0], np.cumsum(fresh)])
    requests = np.full(num_tokens, -1)
    lengths = np.zeros(num_tokens, np.int64)
    slots = np.full(num_tokens, -1)
    taken = lost = 0
    for r, (old, new) in enumerate(zip(past, fresh)):
        for b in range(-(-old // page_size), min(-(-(old + new) // page_size), width)):
            table[r, b] = free_pages[taken] if taken < len(free_pages) else -1
            taken += 1
        for i in range(new):
            t, b = starts[r] + i, (old + i) // page_size
            requests[t], lengths[t] = r, old + i + 1
            if b < width and table[r, b] >= 0:
                slots[t] = table[r, b] * page_size + (old + i) % page_size
            else:
                lost += 1
    return table, starts, requests, lengths, slots, np.array([taken, lost])


def exponent(top):
    """e of the codes x * 2^e of values of at most `top` in magnitude."""
    if top == 0:
        return 100
    if np.isinf(top):
        return -100
    return int(np.clip(6 - np.floor(np.log2(top)), -100, 100))


def page_bounds(rows):
    """Codes [2, dim] and scale of the keys [rows, dim] of one page and head."""
    with np.errstate(all="ignore"):
        nan = np.isnan(rows)
        low = np.where(nan, np.inf, rows).min(0)
        high = np.where(nan, -np.inf, rows).max(0)
        low, high = np.where(nan.all(0), 0, low), np.where(nan.all(0), 0, high)
        e = exponent(max(np.abs(low).max(), np.abs(high).max()))
        codes = [np.clip(np.floor(low * 2.0 ** e), -127, 127),
                 np.clip(np.ceil(high * 2.0 ** e), -127, 127)]
    return np.array(codes).astype(np.int64), 2.0 ** -e


def query_codes(q):
    """Codes [2, dim] (negative and positive part) of one group's q [heads, dim]."""
    top = np.nanmax(np.abs(q)) if not np.isnan(q).all() else 0.0
    with np.errstate(all="ignore"):
        x = np.rint(np.clip(q * 2.0 ** exponent(top), -127, 127))
    x = np.where(np.isnan(x), 0, x).astype(np.int64)
    shift = (len(q) - 1).bit_length()
    up, down = np.maximum(x, 0).sum(0), np.maximum(-x, 0).sum(0)
    return np.array([-(down >> shift), up >> shift])


def paged_select(q, codes, scales, table, lengths, page_size, n, requests, first=1, last=1):
    """Pages [tokens, heads, n]: ascending, -1 past the last."""
    pages, heads = codes.shape[:2]
    group = q.shape[1] // heads
    out = np.full((len(q), heads, n), -1)
    for t in range(len(q)):
        r = requests[t]
        if not 0 <= r < len(table):
            continue
        held = min(-(-max(lengths[t], 0) // page_size), table.shape[1])
        for h in range(heads):
            c = query_codes(q[t, h * group:(h + 1) * group])
            b = np.arange(held)
            p = np.asarray(table[r, :held])
            b, p = b[(p >= 0) & (p < pages)], p[(p >= 0) & (p < pages)]
            dots = (c * codes[p, h]).sum((1, 2))
            score = dots.astype(np.float32) * scales[p, h].astype(np.float64)
            score = np.where((b < first) | (b >= held - last), np.inf, score)
            best = np.sort(b[np.argsort(-score, kind="stable")[:n]])
            out[t, h, :len(best)] = best
    return out


def paged_attention(q, keys, values, table, lengths, requests, scale, pages=None):
    """(out, lse, weight): the attention, its logarithm of the sum of
    exponentials, and sum p |v|, what roundings of the weights are measured
    against.  keys, values: [pages, page_size, heads, dim]."""
    count, page_size, heads, _ = keys.shape
    group = q.shape[1] // heads
    out, weight = np.zeros_like(q), np.zeros_like(q)
    lse = np.full(q.shape[:2], -np.inf)
    for t in range(len(q)):
        r = requests[t]
        if not 0 <= r < len(table):
            continue
        length = min(max(lengths[t], 0), table.shape[1] * page_size)
        for h in range(heads):
            listed = range(-(-length // page_size)) if pages is None else pages[t, h]
            k, v = [], []
            for b in listed:
                if b < 0 or b * page_size >= length or not 0 <= table[r, b] < count:
                    continue
                rows = min(page_size, length - b * page_size)
                k.append(keys[table[r, b], :rows, h])
                v.append(values[table[r, b], :rows, h])
            if not k:
                continue
            k, v = np.concatenate(k), np.concatenate(v)
            for i in range(h * group, (h + 1) * group):
                s = scale * (k @ q[t, i])
                e = np.exp(s - s.max())
                lse[t, i] = s.max() + np.log(e.sum())
                out[t, i] = (e @ v) / e.sum()
                weight[t, i] = (e @ np.abs(v)) / e.sum()
    return out, lse, weight

"""The paged key-value cache's operators as a serving loop calls them, for measurement.

Four operators: the page tables of a step (`tables`), the cache's writes (`store`), the
attention of new tokens over a paged cache (`attention`), and the attention over the pages
that an 8-bit score selects for each query (`sparse`).  `run` computes them by elementary
torch operations in 32 bits, or, where `own` is true, by this repository's entry points.
"""

import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn}
FAR = 1 << 30  # sorts behind every page


def listed():
    return [
        # One decoding step of a small batch: every request gets one token.
        {"name": "tables, one token each", "op": "tables", "requests": 64, "page": 16,
         "past": 2000, "fresh": 1},
        # Prompts of many requests enter at once, some behind a cached prefix.
        {"name": "tables, ragged prompts", "op": "tables", "requests": 1000, "page": 64,
         "past": 3000, "fresh": 2000},
        # One decoding step writes one token per request and refreshes its page's bounds.
        {"name": "store, one token each", "op": "store", "requests": 128, "page": 64,
         "past": 4000, "fresh": 1, "heads": 8, "d": 128, "type": "bf16", "cache": "bf16"},
        # Prompts enter an 8-bit cache.
        {"name": "store, prompts in 8 bits", "op": "store", "requests": 13, "page": 64,
         "past": 700, "fresh": 2500, "heads": 8, "d": 128, "type": "bf16", "cache": "e4m3"},
        # The smallest call: two short conversations, where latency counts.
        {"name": "attention, two short", "op": "attention", "requests": 2, "page": 16,
         "longest": 300, "shortest": 100, "heads": 8, "group": 1, "d": 64, "type": "f16",
         "cache": "f16"},
        # An ordinary batch of ragged conversations, some slots of the batch idle.
        {"name": "attention, ragged batch", "op": "attention", "requests": 64, "page": 16,
         "longest": 5000, "shortest": 0, "heads": 8, "group": 4, "d": 128, "type": "bf16",
         "cache": "bf16"},
        # Few requests over very long documents, 8-bit cache: split over the length.
        {"name": "attention, long in 8 bits", "op": "attention", "requests": 3, "page": 64,
         "longest": 200001, "shortest": 60000, "heads": 8, "group": 8, "d": 128, "type": "bf16",
         "cache": "e4m3"},
        # A full batch at the cache's capacity.
        {"name": "attention, full batch", "op": "attention", "requests": 200, "page": 32,
         "longest": 16000, "shortest": 2000, "heads": 4, "group": 16, "d": 128, "type": "f16",
         "cache": "f16"},
        # Decoding with few selected pages over conversations of middle length.
        {"name": "sparse, one token each", "op": "sparse", "requests": 32, "page": 64,
         "longest": 32000, "shortest": 500, "fresh": 1, "heads": 8, "group": 4, "d": 128,
         "n": 16, "type": "bf16", "cache": "bf16"},
        # Decoding over very long documents, 8-bit cache.
        {"name": "sparse, long in 8 bits", "op": "sparse", "requests": 7, "page": 64,
         "longest": 250000, "shortest": 50000, "fresh": 1, "heads": 8, "group": 8, "d": 128,
         "n": 64, "type": "bf16", "cache": "e4m3"},
        # Prompts: every token of a few long prompts selects its own pages.
        {"name": "sparse, prompts", "op": "sparse", "requests": 3, "page": 64,
         "longest": 12000, "shortest": 4000, "fresh": 2048, "heads": 4, "group": 8, "d": 128,
         "n": 16, "type": "bf16", "cache": "bf16"},
        # Short prompts with odd sizes: pages that are no power of two, six heads a group.
        {"name": "sparse, odd prompts", "op": "sparse", "requests": 5, "page": 24,
         "longest": 1500, "shortest": 3, "fresh": 150, "heads": 2, "group": 6, "d": 80,
         "n": 9, "type": "f16", "cache": "f16"},
    ]


def _between(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["tables", "store", "attention", "attention", "sparse", "sparse"])
    case = {"op": op, "page": rng.choice([16, 24, 32, 64, 64, 128])}
    decode = rng.random() < 0.6
    if op == "tables":
        case["requests"] = _between(rng, 1, 1000)
        case["past"] = _between(rng, 10, 4000)
        case["fresh"] = 1 if decode else _between(rng, 2, 2000)
        return case
    case["heads"] = rng.choice([1, 2, 3, 4, 8])
    case["d"] = rng.choice([64, 80, 96, 128, 128, 128, 256])
    case["type"] = rng.choice(["bf16", "bf16", "f16"])
    case["cache"] = rng.choice([case["type"], case["type"], "e4m3"])
    if op == "store":
        case["requests"] = _between(rng, 1, 128)
        case["past"] = _between(rng, 1, 4000)
        case["fresh"] = 1 if decode else _between(rng, 2, max(2, 30000 // case["requests"]))
        return case
    case["group"] = rng.choice([1, 2, 4, 5, 6, 8, 8, 16])
    wide = case["heads"] * case["d"] * 4
    if op == "attention":
        case["longest"] = _between(rng, 1, 200000)
        case["requests"] = _between(rng, 1, min(200, max(1, 2000000000 // (wide * case["longest"]))))
        case["shortest"] = rng.choice([0, 0, 1 + case["longest"] // 20, case["longest"]])
        return case
    case["n"] = _between(rng, 2, 64)
    if decode:
        case["longest"] = _between(rng, 10, 250000)
        case["requests"] = _between(rng, 1, min(64, max(1, 2000000000 // (wide * case["longest"]))))
        case["fresh"] = 1
    else:
        case["n"] = min(case["n"], 2048 // case["page"])
        case["requests"] = _between(rng, 1, 8)
        case["longest"] = _between(rng, 10, 12000)
        case["fresh"] = _between(rng, 2, 6000 // case["requests"])
    case["shortest"] = rng.choice([0, 1 + case["longest"] // 20, case["longest"]])
    return case


def _ragged(count, low, high, salt):
    """Lengths between low and high, the longest among them; by the sizes alone."""
    r = random.Random(count * 1000003 + high * 101 + low * 7 + salt)
    got = [round(low + (high - low) * r.random() ** 2) for _ in range(count)]
    got[r.randrange(count)] = high
    return got


def _lengths(case):
    """Cached tokens and new ones of every request."""
    n = case["requests"]
    if case["op"] in ("tables", "store"):
        past = _ragged(n, 0, case["past"], 1)
    else:
        past = _ragged(n, case["shortest"], case["longest"], 2)
    fresh = case.get("fresh", 0)
    if fresh > 1:
        return past, _ragged(n, 0 if n > 4 else 1, fresh, 3)
    return past, [fresh] * n


def _ceil(a, b):
    return -(-a // b)


def _pages(case, gen):
    """A table of pages in no order, its page count, and the pages that are left."""
    past, fresh = _lengths(case)
    held = [_ceil(a + b, case["page"]) for a, b in zip(past, fresh)]
    width = max(held) + 3
    count = sum(held) + 5
    order = torch.randperm(count, generator=gen, device="cuda").int()
    at = torch.tensor(held, device="cuda")
    begin = at.cumsum(0) - at
    column = torch.arange(width, device="cuda")
    index = (begin[:, None] + column).clamp(max=count - 1)
    table = torch.where(column < at[:, None], order[index], -1).int()
    return table, count, order[sum(held):]


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)


def _cast(x, kind):
    return x.to(TYPES[kind])


def _bounds(keys):
    """Codes and scales of pages [pages, P, heads, d], all of their rows in use."""
    low, high = keys.float().amin(1), keys.float().amax(1)
    top = torch.maximum(low.abs(), high.abs()).amax(-1)
    e = (7 - torch.frexp(top).exponent).clamp(-100, 100)
    by = torch.ldexp(torch.ones_like(top), e)[..., None]
    codes = torch.stack([(low * by).floor().clamp(min=-127), (high * by).ceil().clamp(max=127)], 2)
    return codes.to(torch.int8), 1 / by[..., 0]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    past, fresh = _lengths(case)
    table, count, left = _pages(case, gen)
    page = case["page"]
    state = {"case": case, "table": table, "tokens": sum(fresh)}
    as_int = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    if case["op"] == "tables":
        state["past"], state["fresh"] = as_int(past), as_int(fresh)
        # The pages of the cached tokens stay, the others go back to the free ones.
        column = torch.arange(table.shape[1], device="cuda")
        mine = column < _ceil(state["past"], page)[:, None]
        state["free"] = torch.cat([table[(table >= 0) & ~mine], left]).contiguous()
        state["table"] = torch.where(mine, table, -1).int().contiguous()
        state["padded"] = _ceil(sum(fresh), 64) * 64
        return state
    heads, d = case["heads"], case["d"]
    # Keys of a page lie about a centre of its own, as the keys of one passage do.
    centre = _normal(gen, count, 1, heads, d)
    state["keys"] = torch.empty(count, page, heads, d, dtype=TYPES[case["cache"]], device="cuda")
    state["values"] = torch.empty_like(state["keys"])
    step = max(1, (1 << 26) // (page * heads * d))
    for a in range(0, count, step):
        part = min(step, count - a)
        state["keys"][a:a + part] = _cast(centre[a:a + part] + _normal(gen, part, page, heads, d), case["cache"])
        state["values"][a:a + part] = _cast(_normal(gen, part, page, heads, d), case["cache"])
    eight = case["cache"] == "e4m3"
    state["k_scale"], state["v_scale"] = (0.75, 1.25) if eight else (1.0, 1.0)
    rows = torch.repeat_interleave(torch.arange(len(past), device="cuda"), as_int(fresh).long() if case["op"] != "attention" else 1).int()
    if case["op"] == "attention":
        state["lengths"] = as_int(past)
    else:
        starts = as_int(fresh).cumsum(0) - as_int(fresh)
        at = as_int(past)[rows.long()] + torch.arange(len(rows), device="cuda") - starts[rows.long()]
        state["lengths"] = (at + 1).int()
    state["rows"] = rows
    if case["op"] == "store":
        state["codes"] = torch.zeros(count, heads, 2, d, dtype=torch.int8, device="cuda")
        state["scales"] = torch.zeros(count, heads, device="cuda")
        state["slots"] = table[rows.long(), at // page].long() * page + at % page
        state["k"] = _cast(1.5 * _normal(gen, len(rows), heads, d), case["type"])
        state["v"] = _cast(_normal(gen, len(rows), heads, d), case["type"])
        return state
    # A query looks for one of its request's pages; the tokens about it look for the same.
    group = case["group"]
    run_of = (state["lengths"].long() // 24) * 7919 + rows.long() * 104729
    want = run_of % _ceil(state["lengths"].long(), page).clamp(min=1)
    near = centre[table[rows.long(), want].clamp(min=0).long(), 0]
    q = near[:, :, None] * 0.6 + 0.8 * _normal(gen, len(rows), heads, group, d)
    state["q"] = _cast(q.reshape(len(rows), heads * group, d), case["type"])
    if case["op"] == "sparse":
        state["codes"], state["scales"] = _bounds(state["keys"])
    return state


# ---------------------------------------------------------------- plain forms


def _plain_tables(s):
    past, fresh, table, free, page = s["past"], s["fresh"], s["table"], s["free"], s["case"]["page"]
    width = table.shape[1]
    column = torch.arange(width, device="cuda")
    first = (past + page - 1) // page
    last = ((past + fresh + page - 1) // page).clamp(max=width)
    need = (last - first).clamp(min=0)
    index = (need.cumsum(0) - need)[:, None] + column - first[:, None]
    new = (column >= first[:, None]) & (column < last[:, None])
    got = torch.where(index < len(free), free[index.clamp(0, len(free) - 1)], -1)
    table.copy_(torch.where(new, got, table))
    ends = fresh.cumsum(0)
    t = torch.arange(s["padded"], device="cuda")
    row = (t[:, None] >= ends).sum(1)
    inside = row < len(past)
    row = row.clamp(max=len(past) - 1)
    at = past[row] + t - (ends - fresh)[row]
    held = torch.where(at // page < width, table[row, (at // page).clamp(max=width - 1)], -1).long()
    slots = torch.where(inside & (held >= 0), held * page + at % page, -1)
    lost = (inside & (slots < 0)).sum()
    starts = torch.cat([ends.new_zeros(1), ends]).int()
    return {"table": table, "starts": starts, "requests": torch.where(inside, row, -1).int(),
            "lengths": torch.where(inside, at + 1, 0).int(), "slots": slots,
            "used": torch.stack([need.sum(), lost]).int()}


def _plain_store(s):
    case, slots, page = s["case"], s["slots"], s["case"]["page"]
    for x, cache, scale in ((s["k"], s["keys"], s["k_scale"]), (s["v"], s["values"], s["v_scale"])):
        x = x.float() * (1 / scale)  # the reciprocal in 32 bits, then one product
        if case["cache"] == "e4m3":
            x = x.clamp(-448, 448)
        cache[slots // page, slots % page] = x.to(cache.dtype)
    # The bounds of every page that got a row, over its rows up to the last one.
    where = torch.cat([slots // page, slots.new_full((1,), -1)])
    ends = slots[where[:-1] != where[1:]]
    keys = s["keys"][ends // page].float()
    used = (torch.arange(page, device="cuda") <= (ends % page)[:, None])[:, :, None, None]
    low = torch.where(used, keys, math.inf).amin(1)
    high = torch.where(used, keys, -math.inf).amax(1)
    top = torch.maximum(low.abs(), high.abs()).amax(-1)
    e = (7 - torch.frexp(top).exponent).clamp(-100, 100)
    by = torch.ldexp(torch.ones_like(top), e)[..., None]
    s["codes"][ends // page, :, 0] = (low * by).floor().clamp(min=-127).to(torch.int8)
    s["codes"][ends // page, :, 1] = (high * by).ceil().clamp(max=127).to(torch.int8)
    s["scales"][ends // page] = 1 / by[..., 0]
    return {"keys": s["keys"], "values": s["values"], "codes": s["codes"], "scales": s["scales"]}


def _softmax_sum(scores, values):
    """Attention by masked scores [..., g, L] over values [..., L, d], and log sums."""
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = torch.where(total > 0, (p @ values) / total, 0.0)
    return out, (top + torch.log(total))[..., 0]


def _plain_attention(s):
    case, lengths, q = s["case"], s["lengths"], s["q"]
    heads, d, page = case["heads"], case["d"], case["page"]
    pages = s["table"][:, :max(1, _ceil(case["longest"], page))].clamp(min=0).long()
    keys = s["keys"][pages].float().flatten(1, 2).permute(0, 2, 3, 1)
    values = s["values"][pages].float().flatten(1, 2).permute(0, 2, 1, 3)
    scores = (q.float().view(len(q), heads, -1, d) @ keys) * (s["k_scale"] / math.sqrt(d))
    inside = torch.arange(scores.shape[-1], device="cuda") < lengths[:, None, None, None]
    out, lse = _softmax_sum(torch.where(inside, scores, -math.inf), torch.where(inside.transpose(2, 3), values, 0.0))
    return {"out": (out * s["v_scale"]).to(q.dtype).view_as(q), "lse": lse.reshape(len(q), -1)}


def _plain_select(s, q, rows, lengths):
    case = s["case"]
    group, page, n = case["group"], case["page"], case["n"]
    x = q.float().view(len(q), case["heads"], group, case["d"])
    top = x.abs().amax((2, 3), keepdim=True)
    e = (7 - torch.frexp(top).exponent).clamp(-100, 100)
    c = torch.round(x * torch.ldexp(torch.ones_like(top), e)).clamp(-127, 127)
    shift = 1 << (group - 1).bit_length()
    up = (c.clamp(min=0).sum(2) / shift).floor()
    down = -((-c).clamp(min=0).sum(2) / shift).floor()
    pages = s["table"][rows]
    codes = s["codes"][pages.clamp(min=0).long()].float().permute(0, 2, 3, 4, 1)
    dots = (down[:, :, None] @ codes[:, :, 0] + up[:, :, None] @ codes[:, :, 1])[:, :, 0]
    scores = dots * s["scales"][pages.clamp(min=0).long()].transpose(1, 2)
    column = torch.arange(pages.shape[1], device="cuda")
    held = ((lengths + page - 1) // page)[:, None]
    forced = (column < 1) | (column >= held - 1)
    scores = torch.where(forced[:, None], math.inf, scores)
    inside = ((column < held) & (pages >= 0))[:, None]
    best = torch.sort(torch.where(inside, scores, -math.inf), dim=-1, descending=True, stable=True)[1][..., :n]
    best = torch.where(inside.expand_as(scores).gather(-1, best), best, FAR).sort(-1)[0]
    best = torch.nn.functional.pad(best, (0, n - best.shape[-1]), value=FAR)
    return torch.where(best == FAR, -1, best).int()


def _plain_sparse(s):
    case, heads, page = s["case"], s["case"]["heads"], s["case"]["page"]
    head = torch.arange(heads, device="cuda")[None, :, None]
    outs, chosen = [], []
    for q, rows, lengths in zip(s["q"].split(256), s["rows"].long().split(256), s["lengths"].split(256)):
        picked = _plain_select(s, q, rows, lengths)
        at = s["table"][rows[:, None, None], picked.clamp(min=0).long()].clamp(min=0).long()
        keys = s["keys"][at, :, head].float().flatten(2, 3)
        values = s["values"][at, :, head].float().flatten(2, 3)
        where = picked[..., None] * page + torch.arange(page, device="cuda")
        inside = ((picked[..., None] >= 0) & (where < lengths[:, None, None, None])).flatten(2)
        x = q.float().view(len(q), heads, -1, case["d"])
        scores = (x @ keys.transpose(2, 3)) * (s["k_scale"] / math.sqrt(case["d"]))
        out, _ = _softmax_sum(torch.where(inside[:, :, None], scores, -math.inf), values)
        outs.append((out * s["v_scale"]).to(q.dtype).view_as(q))
        chosen.append(picked)
    return {"out": torch.cat(outs), "pages": torch.cat(chosen)}


# ---------------------------------------------------------------- the entry points


def _own(s):
    import mlxvs_b200 as mv

    case, op = s["case"], s["case"]["op"]
    if op == "tables":
        t = mv.paged_tables(s["past"], s["fresh"], s["table"], s["free"], case["page"], s["padded"])
        return {"table": s["table"], "starts": t.starts, "requests": t.requests,
                "lengths": t.lengths, "slots": t.slots, "used": t.used}
    if op == "store":
        mv.paged_store(s["k"], s["v"], s["slots"], s["keys"], s["values"], s["codes"], s["scales"],
                       k_scale=s["k_scale"], v_scale=s["v_scale"])
        return {"keys": s["keys"], "values": s["values"], "codes": s["codes"], "scales": s["scales"]}
    if op == "attention":
        out, lse = mv.paged_attention(s["q"], s["keys"], s["values"], s["table"], s["lengths"],
                                      k_scale=s["k_scale"], v_scale=s["v_scale"], return_lse=True)
        return {"out": out, "lse": lse}
    pages = mv.paged_select(s["q"], s["codes"], s["scales"], s["table"], s["lengths"], case["page"],
                            case["n"], requests=s["rows"])
    out = mv.paged_attention(s["q"], s["keys"], s["values"], s["table"], s["lengths"], pages=pages,
                             requests=s["rows"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    return {"out": out, "pages": pages}


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "tables":
        return _plain_tables(state)
    if op == "store":
        return _plain_store(state)
    return _plain_attention(state) if op == "attention" else _plain_sparse(state)


# ---------------------------------------------------------------- exact values and work


def _exact_store(s):
    got = {"codes": None, "scales": None}
    for name, x, scale in (("keys", s["k"], s["k_scale"]), ("values", s["v"], s["v_scale"])):
        flat = s[name].double().flatten(0, 1)
        flat[s["slots"]] = x.double() / scale
        got[name] = flat.view(s[name].shape)
    return got


def exact(case, seed):
    if case["op"] == "tables":
        return None
    s = prepare(case, seed)
    if case["op"] == "store":
        return _exact_store(s)
    past, fresh = _lengths(case)
    page, heads, group, d = case["page"], case["heads"], case["group"], case["d"]
    q = s["q"].double().view(-1, heads, group, d) * (s["k_scale"] / math.sqrt(d))
    out, lse = torch.zeros_like(q), torch.full_like(q[..., 0], -math.inf)
    begin = 0
    for r, old in enumerate(past):
        new = fresh[r] if case["op"] == "sparse" else 1
        held = s["table"][r, :_ceil(old + (new if case["op"] == "sparse" else 0), page)].long()
        if not new or not len(held):
            begin += new
            continue
        for h in range(heads):
            keys = s["keys"][held][:, :, h].double().reshape(-1, d)
            values = s["values"][held][:, :, h].double().reshape(-1, d)
            for a in range(begin, begin + new, 512):
                b = min(a + 512, begin + new)
                x = q[a:b, h]
                scores = torch.einsum("tgd,ld->tgl", x, keys)
                seen = s["lengths"][a:b].long()[:, None]
                mask = torch.arange(len(keys), device="cuda") < seen
                if case["op"] == "sparse":
                    mask = mask & _exact_pages(s, a, b, h, held).repeat_interleave(page, 1)
                scores = scores.masked_fill(~mask[:, None], -math.inf)
                lse[a:b, h] = torch.logsumexp(scores, -1)
                shifted = torch.exp(scores - lse[a:b, h].clamp(min=-1e300)[..., None])
                out[a:b, h] = torch.einsum("tgl,ld->tgd", shifted, values) * s["v_scale"]
        begin += new
    if case["op"] == "sparse":
        return {"out": out.view(s["q"].shape), "pages": None}
    return {"out": out.view(s["q"].shape), "lse": lse.view(len(out), -1)}


def _exact_pages(s, a, b, h, held):
    """Which of the pages `held` tokens a to b of key head h select, in whole numbers."""
    case = s["case"]
    group, page = case["group"], case["page"]
    x = s["q"][a:b].view(b - a, case["heads"], group, case["d"])[:, h].double()
    top = x.abs().amax((1, 2))
    by = torch.exp2((6 - torch.floor(torch.log2(top))).clamp(-100, 100))
    c = torch.round(x * by[:, None, None]).clamp(-127, 127).long()
    bits = (group - 1).bit_length()
    up, down = c.clamp(min=0).sum(1) >> bits, -((-c).clamp(min=0).sum(1) >> bits)
    codes = s["codes"][held, h].double()
    dots = down.double() @ codes[:, 0].T + up.double() @ codes[:, 1].T
    score = dots * s["scales"][held, h].double()
    count = ((s["lengths"][a:b] + page - 1) // page).long()[:, None]
    column = torch.arange(len(held), device="cuda")
    score = torch.where((column < 1) | (column == count - 1), math.inf, score)
    score = torch.where(column < count, score, -math.inf)
    order = torch.argsort(score, dim=1, descending=True, stable=True)
    rank = torch.empty_like(order).scatter_(1, order, column.expand_as(order).contiguous())
    return (rank < case["n"]) & (column < count)


def work(case):
    past, fresh = _lengths(case)
    page, tokens = case["page"], sum(fresh)
    taken = sum(_ceil(a + b, page) - _ceil(a, page) for a, b in zip(past, fresh))
    if case["op"] == "tables":
        return {"bytes": 8 * len(past) + 8 * taken + 16 * tokens + 4 * (len(past) + 1) + 8, "flops": 0}
    heads, d = case["heads"], case["d"]
    size = 1 if case["cache"] == "e4m3" else 2
    if case["op"] == "store":
        touched = sum(_ceil(a + b, page) - a // page for a, b in zip(past, fresh) if b)
        before = sum(a % page for a, b in zip(past, fresh) if b)
        moved = tokens * 2 * (2 + size) + before * size
        return {"bytes": moved * heads * d + 8 * tokens + touched * heads * (2 * d + 4), "flops": 2 * (tokens + before) * heads * d}
    group = case["group"]
    if case["op"] == "attention":
        keys = sum(past)
        return {"bytes": 2 * keys * heads * d * size + len(past) * heads * group * (4 * d + 4),
                "flops": 4 * keys * heads * group * d}
    seen, scored, read = 0, 0, 0
    for a, b in zip(past, fresh):
        mine = [min(case["n"] * page, a + i + 1) for i in range(b)]
        seen += sum(mine)
        read += min(sum(mine), a + b)
        scored += sum(_ceil(a + i + 1, page) for i in range(b))
    pages = sum(_ceil(a + b, page) for a, b in zip(past, fresh) if b)
    return {"bytes": 2 * read * heads * d * size + pages * heads * (2 * d + 4) + tokens * heads * (4 * group * d + 4 * case["n"]),
            "flops": 4 * seen * heads * group * d + 4 * scored * heads * d}

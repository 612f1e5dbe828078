"""GPU tests of the paged cache's operators against the 64-bit oracle.

Whole numbers (tables, slots, codes, selected pages) are equal.  Attention:
with u the unit roundoff of the output's type (bfloat16 2^-8, float16 2^-11),
the output is rounded once (u |o|), the weights p at most once to 16 bits (u
sum p |v|), and a score is a float32 sum of dim products, off by at most
2^-23 dim sum |q k| scale, which moves p by twice that: the tolerance is the
sum of the three, computed per element.  The logarithm of the sum moves by a
score's error and float32 roundings of itself."""

import numpy as np
import pytest

import mlxvs_b200 as mv
from oracle import paged as O

pytestmark = pytest.mark.gpu

UNIT = {"bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}


def torch_():
    import torch

    return torch


def dtype(name):
    return getattr(torch_(), name)


def on_gpu(x, kind="int32"):
    return torch_().tensor(np.asarray(x), dtype=dtype(kind), device="cuda")


def wide(x):
    return x.double().cpu().numpy()


def make_cache(rng, pages, page, heads, dim, kind, layout="plain"):
    """Keys and values with the given memory layout."""
    torch = torch_()
    both = []
    for _ in range(2):
        x = torch.from_numpy(rng.standard_normal((pages, page, heads, dim), np.float32))
        both.append(x.cuda().to(dtype(kind)))
    if layout == "heads first":  # [pages, heads, page, dim] in memory
        both = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in both]
    elif layout == "together":  # keys and values of a page side by side
        both = list(torch.stack(both, 1).unbind(1))
    elif layout == "wide rows":  # rows longer than they need be
        pad = 32
        out = []
        for x in both:
            y = torch.zeros(pages, page, heads, dim + pad, dtype=x.dtype, device="cuda")
            y[..., :dim] = x
            out.append(y[..., :dim])
        both = out
    return both


def make_table(rng, lengths, page, pages, extra=2):
    width = max(-(-max(max(lengths), 1) // page), 1) + extra
    table = np.full((len(lengths), width), -1)
    order, at = rng.permutation(pages), 0
    for r, n in enumerate(lengths):
        need = -(-n // page)
        table[r, :need] = order[at:at + need]
        at += need
    assert at <= pages
    return table


def check_attention(out, lse, q, keys, values, table, lengths, requests, scale, kind, pages=None,
                    k_scale=1.0, v_scale=1.0):
    k, v = wide(keys) * k_scale, wide(values) * v_scale
    k, v = np.nan_to_num(k, nan=0.0), np.nan_to_num(v, nan=0.0)
    want, want_lse, weight = O.paged_attention(wide(q), k, v, table, lengths, requests, scale,
                                               pages)
    dim = q.shape[2]
    size = np.sqrt((wide(q) ** 2).sum(-1)) * np.sqrt((k ** 2).sum(-1).max())
    score_error = 2.0 ** -23 * dim * size * abs(scale)
    u = UNIT[kind]
    tol = u * np.abs(want) + (u + 2 * score_error[..., None] + 2.0 ** -18) * weight + 1e-7
    got = wide(out)
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= tol).all(), np.max(np.abs(got - want) / tol)
    empty = np.isinf(want_lse)
    got = wide(lse)
    assert np.array_equal(got[empty], want_lse[empty])
    assert (wide(out)[empty] == 0).all()
    tol = score_error + 2.0 ** -20 * (1 + np.abs(np.where(empty, 0, want_lse)))
    assert (np.abs(got[~empty] - want_lse[~empty]) <= tol[~empty]).all()


ATTENTION = [
    # lengths, page, heads, group, dim, type, cache, layout
    ([0, 1, 15, 16, 17, 300], 16, 2, 4, 128, "bfloat16", "bfloat16", "plain"),
    ([1], 16, 1, 1, 64, "float16", "float16", "plain"),
    ([33, 0, 700], 24, 3, 6, 80, "float16", "float16", "heads first"),
    ([5, 129], 1, 2, 5, 64, "bfloat16", "bfloat16", "together"),
    ([1000, 2, 63, 64, 65], 64, 2, 8, 256, "bfloat16", "bfloat16", "wide rows"),
    ([4500, 31], 32, 1, 16, 128, "float16", "float16", "plain"),
    ([257, 90], 128, 2, 20, 96, "bfloat16", "bfloat16", "heads first"),
    ([9, 400, 0, 41], 48, 2, 2, 8, "float16", "float16", "plain"),
    ([800, 77], 64, 2, 8, 128, "bfloat16", "float8_e4m3fn", "plain"),
    ([13, 130, 1], 16, 4, 1, 64, "float16", "float8_e4m3fn", "together"),
    ([2050], 24, 1, 7, 256, "bfloat16", "float8_e4m3fn", "heads first"),
    ([350, 100], 7, 2, 33, 16, "float16", "float8_e4m3fn", "wide rows"),
    ([100, 1, 0, 260], 1024, 1, 128, 128, "bfloat16", "bfloat16", "plain"),
    ([20000, 0, 9000, 1, 1], 16, 1, 8, 128, "bfloat16", "bfloat16", "plain"),
]


@pytest.mark.parametrize("lengths,page,heads,group,dim,kind,cache,layout", ATTENTION)
def test_attention(lengths, page, heads, group, dim, kind, cache, layout):
    rng = np.random.default_rng(len(lengths) * 1000 + dim + group)
    pages = sum(-(-n // page) for n in lengths) + 3
    keys, values = make_cache(rng, pages, page, heads, dim, cache, layout)
    table = make_table(rng, lengths, page, pages)
    q = torch_().from_numpy(rng.standard_normal((len(lengths), heads * group, dim)))
    q = (2 * q).cuda().to(dtype(kind))
    ks, vs = (0.5, 1.75) if "8" in cache else (1.0, 1.0)
    # rows past a request's length and pages of nobody hold anything
    used = np.zeros((pages, page), bool)
    for r, n in enumerate(lengths):
        for i in range(n):
            used[table[r, i // page], i % page] = True
    hole = torch_().from_numpy(~used).cuda()[:, :, None, None].expand(keys.shape)
    for x in (keys, values):
        y = x.float()
        y[hole] = float("nan")
        x.copy_(y.to(x.dtype))
    out, lse = mv.paged_attention(q, keys, values, on_gpu(table), on_gpu(lengths), k_scale=ks,
                                  v_scale=vs, return_lse=True)
    assert out.dtype == q.dtype and out.shape == q.shape
    check_attention(out, lse, q, keys, values, table, lengths, range(len(lengths)),
                    dim ** -0.5, kind, k_scale=ks, v_scale=vs)
    again = mv.paged_attention(q, keys, values, on_gpu(table), on_gpu(lengths), k_scale=ks,
                               v_scale=vs)
    assert torch_().equal(out, again)  # a fixed order of sums


def test_attention_masks_and_strides():
    """Tokens of one request and of none, holes in the table, lengths past
    the table, strided queries, another scale, no log sums."""
    rng = np.random.default_rng(3)
    page, heads, group, dim = 16, 2, 4, 128
    keys, values = make_cache(rng, 20, page, heads, dim, "bfloat16")
    table = make_table(rng, [100, 60, 16], page, 20, extra=0)
    table[0, 2] = -1
    table[0, 4] = 20  # beyond the cache
    table[1, 0] = 99999
    requests = [0, 0, 1, -1, 3, 2, 1, 0]
    lengths = [100, 33, 60, 50, 50, 500, 10, -4]
    q = torch_().from_numpy(rng.standard_normal((len(lengths), dim, heads * group + 3)))
    q = q.cuda().to(dtype("bfloat16")).permute(0, 2, 1).contiguous()[:, 1:-2]
    assert not q.is_contiguous()
    out, lse = mv.paged_attention(q, keys, values, on_gpu(table), on_gpu(lengths), scale=0.3,
                                  requests=on_gpu(requests), return_lse=True)
    check_attention(out, lse, q, keys, values, table, lengths, requests, 0.3, "bfloat16")
    # no tokens, and tokens with an empty table
    none = mv.paged_attention(q[:0], keys, values, on_gpu(table), on_gpu(lengths[:0]))
    assert none.shape == (0, heads * group, dim)
    bare = mv.paged_attention(q, keys, values, on_gpu(np.zeros((8, 0))), on_gpu([5] * 8))
    assert (bare == 0).all()


def test_attention_extreme_scores():
    """Very large and very small scores, NaN and infinite rows."""
    torch = torch_()
    rng = np.random.default_rng(4)
    keys, values = make_cache(rng, 8, 16, 1, 64, "bfloat16")
    table = np.arange(8).reshape(2, 4)
    q = torch.randn(2, 2, 64, device="cuda").bfloat16()
    for factor in (1e4, 1e-4):
        x = (q * factor).bfloat16()
        out, lse = mv.paged_attention(x, keys, values, on_gpu(table), on_gpu([64, 50]),
                                      return_lse=True)
        check_attention(out, lse, x, keys, values, table, [64, 50], [0, 1], 0.125, "bfloat16")
    keys[table[0, 1], 3, 0, 5] = float("nan")
    out, lse = mv.paged_attention(q, keys, values, on_gpu(table), on_gpu([64, 50]),
                                  return_lse=True)
    assert out[0].isnan().all() and out[1].isfinite().all()
    assert lse[0].isnan().all() and lse[1].isfinite().all()


def test_attention_offsets_past_32_bits():
    """Pages whose first element is past 2^31 elements of the cache."""
    torch = torch_()
    page, heads, dim = 64, 4, 128
    count = (1 << 31) // (page * heads * dim) + 40
    keys = torch.empty(count, page, heads, dim, dtype=dtype("float8_e4m3fn"), device="cuda")
    values = torch.empty_like(keys)
    rng = np.random.default_rng(5)
    ids = np.array([count - 1, 3, count - 20, count - 7])
    small = make_cache(rng, 4, page, heads, dim, "float8_e4m3fn")
    for big, x in zip((keys, values), small):
        big.view(torch.uint8)[torch.from_numpy(ids).cuda()] = x.view(torch.uint8)
    q = torch.randn(1, 8, dim, device="cuda").bfloat16()
    out, lse = mv.paged_attention(q, keys, values, on_gpu(ids[None]), on_gpu([250]),
                                  return_lse=True)
    check_attention(out, lse, q, *small, np.arange(4)[None], [250], [0], dim ** -0.5, "bfloat16")
    k = torch.randn(3, heads, dim, device="cuda").bfloat16()
    slots = torch.tensor([(count - 3) * page + i for i in (5, 6, 7)], device="cuda")
    mv.paged_store(k, k, slots, keys, values)
    assert torch.equal(keys[count - 3, 5:8].float(), k.to(keys.dtype).float())


SELECTED = [
    ([700, 0, 50, 1], [3, 0, 40, 1], 16, 2, 4, 128, 5, "bfloat16", "bfloat16", "plain"),
    ([900, 300], [70, 33], 24, 2, 6, 80, 9, "float16", "float16", "heads first"),
    ([2000, 64, 65], [1, 1, 1], 64, 3, 8, 128, 7, "bfloat16", "float8_e4m3fn", "plain"),
    ([600], [130], 32, 1, 16, 64, 4, "float16", "float16", "together"),
    ([500, 20], [100, 20], 16, 2, 1, 256, 6, "bfloat16", "bfloat16", "wide rows"),
    ([300, 700], [65, 17], 16, 1, 20, 96, 30, "float16", "float8_e4m3fn", "plain"),
    ([4000], [1], 1, 2, 3, 64, 256, "bfloat16", "bfloat16", "plain"),
    ([1500, 1400], [200, 50], 128, 2, 8, 128, 3, "bfloat16", "bfloat16", "plain"),
    ([300, 31], [33, 31], 8, 2, 4, 8, 6, "float16", "float16", "plain"),
    ([333], [1], 24, 1, 3, 24, 11, "bfloat16", "bfloat16", "heads first"),
    # enough tokens that tiles of them share the pages
    ([900, 400], [380, 220], 64, 8, 8, 128, 5, "bfloat16", "bfloat16", "plain"),
    ([777, 5, 333], [300, 5, 290], 24, 8, 6, 80, 7, "float16", "float16", "heads first"),
    ([1001], [601], 100, 8, 3, 64, 4, "float16", "float8_e4m3fn", "together"),
    ([500, 300], [200, 90], 16, 4, 12, 256, 9, "bfloat16", "bfloat16", "wide rows"),
    ([640], [300], 48, 4, 20, 128, 6, "bfloat16", "float8_e4m3fn", "heads first"),
    ([2500], [560], 1024, 8, 2, 16, 2, "float16", "float8_e4m3fn", "plain"),
    ([400, 300], [310, 250], 32, 8, 1, 256, 3, "bfloat16", "float8_e4m3fn", "plain"),
    ([20000], [600], 16, 8, 4, 64, 40, "float16", "float16", "plain"),
]


@pytest.mark.parametrize("lengths,fresh,page,heads,group,dim,n,kind,cache,layout", SELECTED)
def test_select_and_sparse_attention(lengths, fresh, page, heads, group, dim, n, kind, cache,
                                     layout):
    """The last `fresh` tokens of each request attend to n pages each."""
    torch = torch_()
    rng = np.random.default_rng(dim + n)
    pages = sum(-(-x // page) for x in lengths) + 3
    keys, values = make_cache(rng, pages, page, heads, dim, cache, layout)
    table = make_table(rng, lengths, page, pages)
    used = np.ones(pages, int) * page
    for r, x in enumerate(lengths):
        if x % page:
            used[table[r, x // page]] = x % page
    k = wide(keys)
    bounds = [[O.page_bounds(k[p, :used[p], h]) for h in range(heads)] for p in range(pages)]
    codes = np.array([[b[0] for b in x] for x in bounds])
    scales = np.array([[b[1] for b in x] for x in bounds])
    requests = np.repeat(np.arange(len(lengths)), fresh)
    seen = np.concatenate([np.arange(x - f, x) + 1 for x, f in zip(lengths, fresh)])
    q = 2 * torch.from_numpy(rng.standard_normal((len(seen), heads * group, dim)))
    q = q.cuda().to(dtype(kind))
    args = (on_gpu(codes, "int8"), on_gpu(scales, "float32"), on_gpu(table), on_gpu(seen), page, n)
    got = mv.paged_select(q, *args, requests=on_gpu(requests))
    want = O.paged_select(wide(q), codes, scales, table, seen, page, n, requests)
    assert np.array_equal(got.cpu().numpy(), want)
    out, lse = mv.paged_attention(q, keys, values, on_gpu(table), on_gpu(seen), pages=got,
                                  requests=on_gpu(requests), return_lse=True)
    check_attention(out, lse, q, keys, values, table, seen, requests, dim ** -0.5, kind, want)
    again = mv.paged_attention(q, keys, values, on_gpu(table), on_gpu(seen), pages=got,
                               requests=on_gpu(requests))
    assert torch.equal(out, again)


@pytest.mark.parametrize("tokens,heads", [(45, 2), (700, 8)])
def test_sparse_attention_masks(tokens, heads):
    """Lists with gaps, of nothing, beyond the length and the table's holes;
    tokens of several requests side by side in any order; rows that only the
    later tokens see and that hold infinities and NaN."""
    rng = np.random.default_rng(8)
    page, group, dim, n = 16, 8, 128, 6
    keys, values = make_cache(rng, 40, page, heads, dim, "bfloat16")
    table = make_table(rng, [200, 150, 90], page, 40, extra=0)
    table[1, 3] = -1
    requests = rng.integers(-1, 4, tokens)
    lengths = rng.integers(0, 210, tokens)
    pages = np.full((tokens, heads, n), -1)
    for t in range(tokens):
        for h in range(heads):
            m = rng.integers(0, n + 1)
            pages[t, h, rng.permutation(n)[:m]] = rng.permutation(table.shape[1])[:m]
    pages[7] = -1
    q = torch_().from_numpy(rng.standard_normal((tokens, heads * group, dim))).cuda().bfloat16()
    args = (on_gpu(table), on_gpu(lengths))
    more = dict(pages=on_gpu(pages), requests=on_gpu(requests), return_lse=True)
    out, lse = mv.paged_attention(q, keys, values, *args, **more)
    check_attention(out, lse, q, keys, values, table, lengths, requests, dim ** -0.5, "bfloat16",
                    pages)
    # row 105 of the first request: only tokens that see it may change
    at = table[0, 105 // page], 105 % page
    keys[at] = float("nan")
    values[at] = float("inf")
    out2, _ = mv.paged_attention(q, keys, values, *args, **more)
    sees = np.zeros((tokens, heads), bool)
    for t in range(tokens):
        for h in range(heads):
            sees[t, h] = requests[t] == 0 and lengths[t] > 105 and 105 // page in pages[t, h]
    assert sees.any()
    sees = on_gpu(sees, "bool")[:, :, None, None]
    a, b = (x.view(tokens, heads, group, dim) for x in (out, out2))
    assert torch_().equal(a.masked_fill(sees, 0), b.masked_fill(sees, 0))
    assert b.masked_select(sees).isnan().all()


def test_select_ties_forced_pages_and_odd_queries():
    torch = torch_()
    page, n = 16, 5
    table = np.arange(40)[None].repeat(6, 0)
    table[5, 3] = -1
    codes = torch.ones(40, 1, 2, 64, dtype=torch.int8, device="cuda")
    scales = torch.ones(40, 1, device="cuda")
    q = torch.ones(6, 3, 64, device="cuda").half()
    q[1] = 0
    q[2, 0, 0] = float("nan")
    q[3, 1, 5] = float("inf")
    q[4] = -q[4]
    lengths = [640, 639, 100, 64, 600, 640]
    run = lambda **kw: mv.paged_select(q, codes, scales, on_gpu(table), on_gpu(lengths), page, n,  # noqa: E731
                                       **kw).cpu().numpy()
    for first, last in ((1, 1), (0, 0), (2, 3), (0, 5), (5, 0)):
        want = O.paged_select(wide(q), codes.cpu().numpy().astype(int), scales.cpu().numpy(),
                              table, lengths, page, n, range(6), first, last)
        assert np.array_equal(run(first=first, last=last), want)
    assert run()[0, 0].tolist() == [0, 1, 2, 3, 39]
    assert run()[3, 0].tolist() == [0, 1, 2, 3, -1]
    empty = mv.paged_select(q[:0], codes, scales, on_gpu(table), on_gpu(lengths[:0]), page, n)
    assert empty.shape == (0, 1, n)


def test_select_of_tokens_in_any_order():
    """Tokens of several requests and of none, interleaved."""
    rng = np.random.default_rng(13)
    tokens, heads, group, dim, page, n = 61, 3, 5, 96, 16, 6
    codes = np.sort(rng.integers(-127, 128, (70, heads, 2, dim)), 2)
    scales = 2.0 ** rng.integers(-3, 3, (70, heads))
    table = rng.integers(-2, 72, (4, 30))  # holes, and pages beyond the cache
    requests = rng.integers(-1, 5, tokens)
    lengths = rng.integers(-3, 600, tokens)
    q = torch_().from_numpy(rng.standard_normal((tokens, heads * group, dim))).cuda().half()
    got = mv.paged_select(q, on_gpu(codes, "int8"), on_gpu(scales, "float32"), on_gpu(table),
                          on_gpu(lengths), page, n, requests=on_gpu(requests), first=2, last=2)
    want = O.paged_select(wide(q), codes, scales, table, lengths, page, n, requests, 2, 2)
    assert np.array_equal(got.cpu().numpy(), want)


def test_strides_of_single_elements_and_given_streams():
    """A dimension of one element may have any stride; stream= takes a torch
    stream or a handle."""
    torch = torch_()
    rng = np.random.default_rng(14)
    keys, values = make_cache(rng, 3, 16, 1, 64, "float16")
    table, lengths = on_gpu([[2, 0, 1]]), on_gpu([40])
    q = torch.randn(1, 1, 64, device="cuda").half()
    odd = q.as_strided((1, 1, 64), (3, 5, 1))
    oddk, oddv = (x.as_strided(x.shape, (x.stride(0), x.stride(1), 7, 1)) for x in (keys, values))
    want = mv.paged_attention(q, keys, values, table, lengths)
    assert torch.equal(mv.paged_attention(odd, oddk, oddv, table, lengths), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for stream in (side, side.cuda_stream):
        got = mv.paged_attention(q, keys, values, table, lengths, stream=stream)
        side.synchronize()
        assert torch.equal(got, want)
    t = mv.paged_tables(on_gpu([5]), on_gpu([2]), table, on_gpu([1]), 16, 2, stream=side)
    side.synchronize()
    assert t.slots.tolist() == [2 * 16 + 5, 2 * 16 + 6]


def test_select_many_pages():
    """More candidates than threads, scores of both signs and wide scales."""
    rng = np.random.default_rng(10)
    count = 12001
    codes = np.sort(rng.integers(-127, 128, (count, 2, 2, 128)), 2)
    scales = 2.0 ** rng.integers(-30, 30, (count, 2))
    table = rng.permutation(count)[None].repeat(3, 0)
    q = torch_().from_numpy(rng.standard_normal((3, 8, 128))).cuda().bfloat16()
    lengths = [count * 16, 5000 * 16 - 3, 17 * 16]
    for n in (1, 2, 16, 200, 256):
        first = min(1, n - 1)
        got = mv.paged_select(q, on_gpu(codes, "int8"), on_gpu(scales, "float32"), on_gpu(table),
                              on_gpu(lengths), 16, n, first=first)
        want = O.paged_select(wide(q), codes, scales, table, lengths, 16, n, range(3), first)
        assert np.array_equal(got.cpu().numpy(), want)


STORED = [
    ([0, 5, 15, 16, 40], [1, 1, 1, 1, 1], 16, 2, 128, "bfloat16", "bfloat16", "plain"),
    ([0, 30, 7], [100, 3, 0], 24, 3, 80, "float16", "float16", "heads first"),
    ([3, 64, 100], [70, 64, 29], 64, 2, 256, "bfloat16", "float8_e4m3fn", "together"),
    ([10], [300], 1, 1, 64, "float16", "float8_e4m3fn", "plain"),
    ([1000, 1], [30, 1030], 1024, 1, 16, "bfloat16", "bfloat16", "wide rows"),
    ([5] * 70, [2] * 70, 48, 8, 128, "bfloat16", "bfloat16", "plain"),
]


@pytest.mark.parametrize("past,fresh,page,heads,dim,kind,cache,layout", STORED)
def test_store(past, fresh, page, heads, dim, kind, cache, layout):
    torch = torch_()
    rng = np.random.default_rng(dim + page)
    held = [a + b for a, b in zip(past, fresh)]
    pages = sum(-(-x // page) for x in held) + 2
    keys, values = make_cache(rng, pages, page, heads, dim, cache, layout)
    table = make_table(rng, held, page, pages)
    slots = np.concatenate([[table[r, i // page] * page + i % page for i in range(a, a + b)]
                            for r, (a, b) in enumerate(zip(past, fresh))]).astype(int)
    ks, vs = (0.3, 7.0) if "8" in cache else (1.0, 1.0)
    k, v = (torch.from_numpy(3 * rng.standard_normal((len(slots), heads, dim))).cuda().to(
        dtype(kind)) for _ in range(2))
    k[0, 0, :4] = torch.tensor([0.0, -0.0, 1e4, -1e4])
    skipped = len(slots) // 2 if len(slots) > 6 else -1
    if skipped >= 0:
        slots[skipped] = -1
    codes = torch.full((pages, heads, 2, dim), 77, dtype=torch.int8, device="cuda")
    scales = torch.full((pages, heads), -1.0, device="cuda")
    before = keys.clone(), values.clone()
    mv.paged_store(k, v, on_gpu(slots, "int64"), keys, values, codes, scales, k_scale=ks,
                   v_scale=vs)
    where = torch.from_numpy(slots[slots >= 0]).cuda()
    for x, old, new, scale in ((k, before[0], keys, ks), (v, before[1], values, vs)):
        y = x.float() * float(np.float32(1) / np.float32(scale))
        if "8" in cache:
            y = y.clamp(-448, 448)
        old[where // page, where % page] = y.to(old.dtype)[torch.from_numpy(slots >= 0).cuda()]
        assert torch.equal(old.view(torch.uint8), new.view(torch.uint8))
    last = {}
    for s in slots[slots >= 0]:
        last[s // page] = max(last.get(s // page, 0), s % page)
    k = wide(keys)
    for p in range(pages):
        for h in range(heads):
            if p in last:
                c, s = O.page_bounds(k[p, :last[p] + 1, h])
                assert np.array_equal(codes[p, h].cpu().numpy(), c) and scales[p, h].item() == s
            else:
                assert (codes[p, h] == 77).all() and scales[p, h].item() == -1
    # without bounds: the rows alone
    mv.paged_store(v, v, on_gpu(slots, "int64"), *before, k_scale=vs,
                   v_scale=vs)
    assert torch.equal(before[0][where // page, where % page].view(torch.uint8),
                       before[1][where // page, where % page].view(torch.uint8))


def test_store_bounds_of_special_keys():
    """NaN, infinite, zero and tiny keys; the same page row by row."""
    torch = torch_()
    rng = np.random.default_rng(11)
    keys, values = make_cache(rng, 6, 8, 1, 64, "bfloat16")
    k = torch.from_numpy(rng.standard_normal((48, 1, 64))).cuda().bfloat16()
    k[3, 0, 7] = float("nan")
    k[8:16, 0, 9] = float("nan")
    k[17, 0, 1] = float("inf")
    k[18, 0, 2] = -float("inf")
    k[24:32] = 0
    k[32:40] *= 1e-38
    k[40:48] *= 1e30
    slots = on_gpu(np.arange(48), "int64")
    codes = torch.zeros(6, 1, 2, 64, dtype=torch.int8, device="cuda")
    scales = torch.zeros(6, 1, device="cuda")
    mv.paged_store(k, k, slots, keys, values, codes, scales)
    for p in range(6):
        c, s = O.page_bounds(wide(keys)[p, :, 0])
        assert np.array_equal(codes[p, 0].cpu().numpy(), c) and scales[p, 0].item() == s
    one = torch.zeros_like(codes), torch.zeros_like(scales)
    for i in range(48):
        mv.paged_store(k[i:i + 1], k[i:i + 1], slots[i:i + 1], keys, values, *one)
    assert torch.equal(one[0], codes) and torch.equal(one[1], scales)


TABLES = [
    ([0, 5, 16, 31, 32], [1, 1, 1, 1, 1], 16, 0, 99),
    ([0, 0, 100, 3], [50, 0, 7, 1000], 24, 5, 99),
    ([7], [0], 64, 3, 9),
    ([1, 2, 3], [40, 40, 40], 8, 0, 7),       # the free list ends
    ([100, 0], [300, 300], 16, 0, 999),       # the table is too narrow
    ([0] * 3000, [1] * 3000, 16, 100, 3000),
    ([11] * 700 + [0] * 100, [0] * 300 + [9] * 500, 4, 1, 5000),
    ([0, 9000], [5000, 1], 1, 0, 9999),
]


@pytest.mark.parametrize("past,fresh,page,padding,free", TABLES)
def test_tables(past, fresh, page, padding, free):
    torch = torch_()
    rng = np.random.default_rng(page)
    width = max(-(-(a + b) // page) for a, b in zip(past, fresh))
    if past == [100, 0]:
        width = 20
    table = np.full((len(past), width), -7)
    ids = rng.permutation(len(past) * width + free)
    at = 0
    for r, a in enumerate(past):
        need = min(-(-a // page), width)
        table[r, :need] = ids[at:at + need]
        at += need
    if past == [1, 2, 3]:
        table[1, 0] = -1  # a begun page that the table does not hold
    free_pages = ids[at:at + free]
    tokens = sum(fresh) + padding
    want = O.paged_tables(past, fresh, table, free_pages, page, tokens)
    gpu = on_gpu(table)
    for _ in range(2):  # the same again on the table it has filled
        got = mv.paged_tables(on_gpu(past), on_gpu(fresh), gpu, on_gpu(free_pages), page, tokens)
        assert np.array_equal(gpu.cpu().numpy(), want[0])
        for x, y in zip(got, want[1:]):
            assert np.array_equal(x.cpu().numpy(), y)
    assert got.slots.dtype == torch.int64


def test_tables_of_no_requests():
    got = mv.paged_tables(on_gpu([]), on_gpu([]), on_gpu(np.zeros((0, 4))), on_gpu([1, 2]), 16, 3)
    assert got.starts.tolist() == [0] and got.used.tolist() == [0, 0]
    assert got.slots.tolist() == [-1] * 3 and got.requests.tolist() == [-1] * 3
    assert got.lengths.tolist() == [0] * 3


def test_a_step_on_another_stream_and_in_a_graph():
    """tables, store, select and attention of a decoding step, on a stream of
    their own and replayed from a CUDA graph with new inputs."""
    torch = torch_()
    rng = np.random.default_rng(12)
    page, heads, group, dim, n, requests = 16, 2, 4, 64, 4, 5
    past = np.array([0, 15, 16, 100, 333])
    keys, values = make_cache(rng, 60, page, heads, dim, "float16")
    codes = torch.zeros(60, heads, 2, dim, dtype=torch.int8, device="cuda")
    scales = torch.zeros(60, heads, device="cuda")
    host_table = make_table(rng, list(past), page, 50)
    for r in range(requests):  # the bounds of what is there
        for b in range(-(-past[r] // page)):
            for h in range(heads):
                rows = min(page, past[r] - b * page)
                c, s = O.page_bounds(wide(keys)[host_table[r, b], :rows, h])
                codes[host_table[r, b], h] = on_gpu(c, "int8")
                scales[host_table[r, b], h] = s
    used = set(host_table[host_table >= 0])
    free = on_gpu([p for p in range(60) if p not in used])
    table, old, fresh = on_gpu(host_table), on_gpu(past), on_gpu([1] * requests)
    k, v = (torch.randn(requests, heads, dim, device="cuda").half() for _ in range(2))
    q = torch.randn(requests, heads * group, dim, device="cuda").half()

    def step():
        t = mv.paged_tables(old, fresh, table, free, page, requests)
        mv.paged_store(k, v, t.slots, keys, values, codes, scales)
        p = mv.paged_select(q, codes, scales, table, t.lengths, page, n, requests=t.requests)
        out, lse = mv.paged_attention(q, keys, values, table, t.lengths, requests=t.requests,
                                      pages=p, return_lse=True)
        return t, p, out, lse

    def check(t, p, out, lse):
        seen = old.cpu().numpy() + 1
        assert np.array_equal(t.lengths.cpu().numpy(), seen)
        want = O.paged_select(wide(q), codes.cpu().numpy().astype(int), scales.cpu().numpy(),
                              table.cpu().numpy(), seen, page, n, range(requests))
        assert np.array_equal(p.cpu().numpy(), want)
        check_attention(out, lse, q, keys, values, table.cpu().numpy(), seen, range(requests),
                        dim ** -0.5, "float16", want)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    check(*got)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(2):
        k.normal_(), v.normal_(), q.normal_()
        graph.replay()
        torch.cuda.synchronize()
        check(*got)
    mv.synchronize()


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
def test_example(cache):
    """The decoding example: with all pages selected the sparse attention is
    the whole one; with few, part of its weight."""
    import importlib.util
    import os

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples",
                        "paged_decode.py")
    spec = importlib.util.spec_from_file_location("paged_decode", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    few = example.run(requests=5, steps=3, passage_tokens=100, pages_seen=3, cache=cache)
    assert len(few) == 4 and all(0.1 < s < 1.0 for s in few)
    every = example.run(requests=5, steps=3, passage_tokens=100, pages_seen=16, cache=cache)
    # both sum the same weights, in another order: float32 roundings
    assert all(abs(s - 1.0) < 1e-4 for s in every)

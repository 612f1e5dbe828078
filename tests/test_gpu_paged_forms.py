"""GPU tests that reach every form of the paged attention's kernels (types,
head dimensions, heads a key head, whole cache or selected pages, prompts), the
selection's tiles on clusters of blocks, and calls with cut rows and with prompts
in a CUDA graph.  Tolerances as in test_gpu_paged.py."""

import numpy as np
import pytest

import mlxvs_b200 as mv
from oracle import paged as O
from tests.test_gpu_paged import (
    check_attention, dtype, make_cache, make_table, on_gpu, torch_, wide,
)

pytestmark = pytest.mark.gpu

TYPES = [("bfloat16", "bfloat16"), ("float16", "float16"), ("bfloat16", "float8_e4m3fn"),
         ("float16", "float8_e4m3fn")]


def lists_of_pages(rng, lengths, requests, page, heads, n):
    """Up to n pages of each token and head, ascending, -1 past the last."""
    got = np.full((len(lengths), heads, n), -1)
    for t, x in enumerate(lengths):
        held = -(-x // page)
        for h in range(heads):
            m = min(n, held)
            got[t, h, :m] = np.sort(rng.permutation(held)[:m])
    return got


@pytest.mark.parametrize("selected", [False, True])
@pytest.mark.parametrize("group", [3, 8, 11, 16])
@pytest.mark.parametrize("dim", [48, 64, 112, 128, 208, 256])
@pytest.mark.parametrize("kind,cache", TYPES)
def test_attention_forms(kind, cache, dim, group, selected):
    """Rows of one token; tables wide enough that rows are cut and joined."""
    rng = np.random.default_rng(dim + group)
    page, heads, lengths = 16, 2, [1300, 0, 40, 517]
    pages = sum(-(-x // page) for x in lengths) + 2
    keys, values = make_cache(rng, pages, page, heads, dim, cache)
    table = make_table(rng, lengths, page, pages, extra=60)
    q = torch_().from_numpy(2 * rng.standard_normal((4, heads * group, dim))).cuda().to(dtype(kind))
    ks, vs = (0.5, 1.75) if "8" in cache else (1.0, 1.0)
    chosen = lists_of_pages(rng, lengths, range(4), page, heads, 70) if selected else None
    more = dict(pages=on_gpu(chosen)) if selected else {}
    out, lse = mv.paged_attention(q, keys, values, on_gpu(table), on_gpu(lengths), k_scale=ks,
                                  v_scale=vs, return_lse=True, **more)
    check_attention(out, lse, q, keys, values, table, lengths, range(4), dim ** -0.5, kind, chosen,
                    k_scale=ks, v_scale=vs)


@pytest.mark.parametrize("group", [2, 10])
@pytest.mark.parametrize("dim", [32, 128, 224])
@pytest.mark.parametrize("kind,cache", TYPES)
def test_prompt_forms(kind, cache, dim, group):
    """Tiles of a prompt's tokens, with one and with two groups of 8 heads."""
    rng = np.random.default_rng(dim)
    page, heads, tokens, length = 40, 8, 420, 900
    pages = -(-length // page) + 2
    keys, values = make_cache(rng, pages, page, heads, dim, cache)
    table = make_table(rng, [length], page, pages)
    requests, seen = [0] * tokens, np.arange(length - tokens, length) + 1
    q = 2 * rng.standard_normal((tokens, heads * group, dim))
    q = torch_().from_numpy(q).cuda().to(dtype(kind))
    chosen = lists_of_pages(rng, seen, requests, page, heads, 4)
    ks, vs = (0.5, 1.75) if "8" in cache else (1.0, 1.0)
    mv.profile_enable()
    out, lse = mv.paged_attention(q, keys, values, on_gpu(table), on_gpu(seen), k_scale=ks,
                                  v_scale=vs, return_lse=True, pages=on_gpu(chosen),
                                  requests=on_gpu(requests))
    launches = mv.profile_read("paged_prompt")[1]
    mv.profile_enable(False)
    assert launches == 1
    check_attention(out, lse, q, keys, values, table, seen, requests, dim ** -0.5, kind, chosen,
                    k_scale=ks, v_scale=vs)


@pytest.mark.parametrize("width,tokens,heads,group,dim", [
    (200, 9, 2, 4, 128), (200, 60, 1, 3, 64), (500, 60, 2, 5, 96), (500, 17, 3, 1, 256),
    (1100, 33, 2, 8, 128), (2000, 60, 1, 2, 80), (6000, 12, 4, 4, 64)])
def test_select_tiles_on_clusters(width, tokens, heads, group, dim):
    """Few tokens of several requests in any order over wide tables with holes:
    clusters of 2, 4 and 8 blocks share the pages of a tile of 8 tokens."""
    rng = np.random.default_rng(width + tokens)
    page, n, count = 16, 12, 300
    codes = np.sort(rng.integers(-127, 128, (count, heads, 2, dim)), 2)
    scales = 2.0 ** rng.integers(-3, 3, (count, heads))
    table = rng.integers(-2, count + 2, (4, width))  # holes, and pages beyond the cache
    q = torch_().from_numpy(rng.standard_normal((tokens, heads * group, dim))).cuda().bfloat16()
    for rows in (4, 1):
        requests = rng.integers(-1, rows + 1, tokens)
        lengths = rng.integers(-3, width * page + 1, tokens)
        got = mv.paged_select(q, on_gpu(codes, "int8"), on_gpu(scales, "float32"),
                              on_gpu(table[:rows]), on_gpu(lengths), page, n,
                              requests=on_gpu(requests), first=2, last=3)
        want = O.paged_select(wide(q), codes, scales, table[:rows], lengths, page, n, requests, 2,
                              3)
        assert np.array_equal(got.cpu().numpy(), want)


def test_cut_rows_and_prompts_in_a_graph():
    """Scratch, cut rows and their joining, and a prompt, replayed with new
    queries and lengths."""
    torch = torch_()
    rng = np.random.default_rng(31)
    page, heads, group, dim = 32, 4, 4, 64
    top = [3000, 900, 2000]
    pages = sum(-(-x // page) for x in top) + 2
    keys, values = make_cache(rng, pages, page, heads, dim, "float16")
    host = make_table(rng, top, page, pages)
    table = on_gpu(host)
    lengths, tokens = on_gpu(top), 900
    q = torch.zeros(3, heads * group, dim, device="cuda").half()
    pq = torch.zeros(tokens, heads * group, dim, device="cuda").half()
    seen = np.arange(1, tokens + 1)
    requests = [1] * tokens
    chosen = lists_of_pages(rng, seen, requests, page, heads, 5)
    args = dict(requests=on_gpu(requests), pages=on_gpu(chosen))
    plen = on_gpu(seen)

    def step():
        return (*mv.paged_attention(q, keys, values, table, lengths, return_lse=True),
                *mv.paged_attention(pq, keys, values, table, plen, return_lse=True, **args))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for now in (top, [1, 899, 0], [2999, 0, 64]):
        lengths.copy_(on_gpu(now))
        q.normal_(), pq.normal_()
        graph.replay()
        torch.cuda.synchronize()
        check_attention(got[0], got[1], q, keys, values, host, now, range(3), dim ** -0.5,
                        "float16")
        check_attention(got[2], got[3], pq, keys, values, host, seen, requests, dim ** -0.5,
                        "float16", chosen)
    mv.synchronize()


@pytest.mark.parametrize("requests,per,tiles", [(200, 2, 0), (50, 8, 0), (8, 60, 1), (1, 420, 1)])
def test_tokens_a_request_of_the_prompt_kernel(requests, per, tiles):
    """Steps of few tokens a request are not walked as a prompt is, and give
    the same."""
    rng = np.random.default_rng(requests)
    page, heads, group, dim, length = 16, 8, 2, 64, max(100, per)
    pages = requests * -(-length // page) + 2
    keys, values = make_cache(rng, pages, page, heads, dim, "bfloat16")
    table = make_table(rng, [length] * requests, page, pages)
    rows = np.repeat(np.arange(requests), per)
    seen = np.tile(np.arange(length - per, length) + 1, requests)
    q = 2 * rng.standard_normal((len(rows), heads * group, dim))
    q = torch_().from_numpy(q).cuda().to(dtype("bfloat16"))
    chosen = lists_of_pages(rng, seen, rows, page, heads, 3)
    mv.profile_enable()
    out, lse = mv.paged_attention(q, keys, values, on_gpu(table), on_gpu(seen), return_lse=True,
                                  pages=on_gpu(chosen), requests=on_gpu(rows))
    launches = mv.profile_read("paged_prompt")[1]
    mv.profile_enable(False)
    assert launches == tiles
    check_attention(out, lse, q, keys, values, table, seen, rows, dim ** -0.5, "bfloat16", chosen)


@pytest.mark.parametrize("heads,group,page,tokens,length,kind,cache", [
    (1, 2, 16, 3400, 3500, "bfloat16", "bfloat16"),
    (1, 1, 64, 3300, 3300, "float16", "float8_e4m3fn"),
    (8, 2, 1024, 700, 900, "float16", "float16"),  # one page
])
def test_prompts_over_dimensions_of_one(heads, group, page, tokens, length, kind, cache):
    """One key head, or one page: such a dimension's stride may be any."""
    rng = np.random.default_rng(page)
    dim, pages = 64, -(-length // page)
    keys, values = make_cache(rng, pages, page, heads, dim, cache)
    strides = list(keys.stride())
    strides[2 if heads == 1 else 0] = 7
    odd = [x.as_strided(x.shape, strides) for x in (keys, values)]
    table = make_table(rng, [length], page, pages)
    rows, seen = [0] * tokens, np.arange(length - tokens, length) + 1
    q = 2 * rng.standard_normal((tokens, heads * group, dim))
    q = torch_().from_numpy(q).cuda().to(dtype(kind))
    chosen = lists_of_pages(rng, seen, rows, page, heads, 6)
    mv.profile_enable()
    out, lse = mv.paged_attention(q, *odd, on_gpu(table), on_gpu(seen), return_lse=True,
                                  pages=on_gpu(chosen), requests=on_gpu(rows))
    launches = mv.profile_read("paged_prompt")[1]
    mv.profile_enable(False)
    assert launches == 1
    check_attention(out, lse, q, keys, values, table, seen, rows, dim ** -0.5, kind, chosen)

"""GPU tests of the paged cache's operators at the edges of their inputs:
skipped tokens, odd values in what the device reads, several host threads.
Whole numbers are equal; tolerances stand at the tests that have one."""

import numpy as np
import pytest

import mlxvs_b200 as mv
from oracle import paged as O
from tests.test_gpu_paged import UNIT, dtype, make_cache, make_table, on_gpu, torch_, wide

pytestmark = pytest.mark.gpu


# past, fresh, page, heads, dim, type, cache, share of skipped tokens
GAPS = [
    ([3, 64, 100], [70, 64, 29], 64, 2, 128, "bfloat16", "float8_e4m3fn", 0.1),
    ([0, 30, 7], [100, 3, 0], 24, 3, 80, "float16", "float16", 0.5),
    ([1000, 1], [30, 1030], 1024, 1, 16, "bfloat16", "bfloat16", 0.97),
    ([5] * 70, [2] * 70, 48, 8, 128, "bfloat16", "bfloat16", 0.5),
    # chunks of several tokens: 16 at most from 148 * 16 * 16 / 8 tokens on
    ([17, 0, 5], [3000, 2000, 1900], 128, 8, 64, "float16", "float8_e4m3fn", 0.05),
    ([0], [2500], 1, 8, 64, "float16", "float16", 0.3),
]


@pytest.mark.parametrize("past,fresh,page,heads,dim,kind,cache,share", GAPS)
def test_store_with_skipped_tokens(past, fresh, page, heads, dim, kind, cache, share):
    """Any of a page's new tokens may be skipped: the page's bounds cover its
    rows up to the last written one, whatever blocks write them."""
    torch = torch_()
    rng = np.random.default_rng(page + dim)
    held = [a + b for a, b in zip(past, fresh)]
    pages = sum(-(-x // page) for x in held) + 2
    start = make_cache(rng, pages, page, heads, dim, cache)
    table = make_table(rng, held, page, pages)
    slots = np.concatenate([[table[r, i // page] * page + i % page for i in range(a, a + b)]
                            for r, (a, b) in enumerate(zip(past, fresh))]).astype(int)
    slots = np.concatenate([slots, np.full(100, -1)])  # padding
    for _ in range(3):
        at = slots.copy()
        skipped = rng.random(len(at)) < share
        at[skipped] = rng.choice([-1, pages * page, pages * page + 77], skipped.sum())
        k = torch.from_numpy(3 * rng.standard_normal((len(at), heads, dim))).cuda().to(dtype(kind))
        live = (at >= 0) & (at < pages * page)
        where = torch.from_numpy(at[live]).cuda()
        want = start[0].clone()
        want[where // page, where % page] = k[torch.from_numpy(live).cuda()].to(want.dtype)
        last = {}
        for s in at[live]:
            last[s // page] = max(last.get(s // page, 0), s % page)
        rows = wide(want)
        codes = np.full((pages, heads, 2, dim), 77)
        scales = np.full((pages, heads), -1.0)
        for p, row in last.items():
            for h in range(heads):
                codes[p, h], scales[p, h] = O.page_bounds(rows[p, :row + 1, h])
        codes, scales = on_gpu(codes, "int8"), on_gpu(scales, "float32")
        where = on_gpu(at, "int64")
        for _ in range(20):
            keys, values = start[0].clone(), start[1].clone()
            got = torch.full_like(codes, 77), torch.full_like(scales, -1.0)
            mv.paged_store(k, k, where, keys, values, *got)
            assert torch.equal(keys.view(torch.uint8), want.view(torch.uint8))
            assert torch.equal(got[0], codes) and torch.equal(got[1], scales)


def select_case(rng, count, widths, tokens, heads=2, group=4, dim=64):
    """Codes of `count` pages, a table with a row per width and tokens that see
    all of their request's pages (of 16 rows)."""
    codes = np.sort(rng.integers(-127, 128, (count, heads, 2, dim)), 2)
    table = np.full((len(widths), max(widths)), -1)
    for r, w in enumerate(widths):
        table[r, :w] = rng.integers(0, count, w)
    requests = rng.integers(0, len(widths), tokens)
    lengths = np.array(widths)[requests] * 16 - rng.integers(0, 16, tokens)
    q = torch_().from_numpy(rng.standard_normal((tokens, heads * group, dim))).cuda().half()
    return codes, table, requests, lengths, q


@pytest.mark.parametrize("share", [1.0, 0.6])
@pytest.mark.parametrize("widths,tokens", [([40], 1), ([700, 60], 2), ([100, 30, 9], 50)])
def test_select_of_scores_that_are_not_numbers(widths, tokens, share):
    """Scales that are NaN, or infinite where the codes are zero: NaN scores come
    last, lists keep to their n entries."""
    rng = np.random.default_rng(20)
    n = 5
    codes, table, requests, lengths, q = select_case(rng, 300, widths, tokens)
    codes[::7] = 0  # infinite scales times zero
    scales = 2.0 ** rng.integers(-3, 3, (300, 2))
    odd = rng.random(scales.shape) < share
    scales[odd] = np.nan
    scales[::7][odd[::7]] = np.inf
    for first, last in ((1, 1), (0, 0), (5, 0), (2, 3)):
        with np.errstate(all="ignore"):
            want = O.paged_select(wide(q), codes, scales, table, lengths, 16, n, requests, first,
                                  last)
        got = mv.paged_select(q, on_gpu(codes, "int8"), on_gpu(scales, "float32"), on_gpu(table),
                              on_gpu(lengths), 16, n, requests=on_gpu(requests), first=first,
                              last=last)
        assert np.array_equal(got.cpu().numpy(), want)


@pytest.mark.parametrize("widths,tokens", [([40], 1), ([700, 60], 2), ([100, 30, 9], 50)])
def test_select_of_infinite_scores(widths, tokens):
    """Infinite scores of both signs beside finite ones: the largest order bits
    that there are."""
    rng = np.random.default_rng(21)
    codes, table, requests, lengths, q = select_case(rng, 300, widths, tokens)
    codes[codes == 0] = 1
    for share in (0.02, 0.5):
        scales = 2.0 ** rng.integers(-100, 101, (300, 2))
        odd = rng.random(scales.shape) < share
        scales[odd] = rng.choice([np.inf, -np.inf], odd.sum())
        for n in (1, 3, 8):
            with np.errstate(all="ignore"):  # a few dot products are 0: NaN
                want = O.paged_select(wide(q), codes, scales, table, lengths, 16, n, requests, 0,
                                      0)
            got = mv.paged_select(q, on_gpu(codes, "int8"), on_gpu(scales, "float32"),
                                  on_gpu(table), on_gpu(lengths), 16, n,
                                  requests=on_gpu(requests), first=0, last=0)
            assert np.array_equal(got.cpu().numpy(), want)


def test_tables_of_impossible_lengths():
    """Lengths and sums past 2^31 (which the caller rules out): what lies about
    the table stays, slots are in the free pages or -1, requests before the
    impossible one are right."""
    torch = torch_()
    rng = np.random.default_rng(22)
    top = 2 ** 31 - 1
    free = np.arange(50, 150)

    def run(past, fresh, page, width, tokens):
        room = torch.full((3, len(past), width), -9, dtype=torch.int32, device="cuda")
        room[1] = -1
        got = mv.paged_tables(on_gpu(past), on_gpu(fresh), room[1], on_gpu(free), page, tokens)
        mv.synchronize()
        assert (room[0] == -9).all() and (room[2] == -9).all()
        slots = got.slots.cpu().numpy()
        assert ((slots == -1) | ((slots >= 50 * page) & (slots < 150 * page))).all()
        return got, room[1]

    for page in (1, 16, 1000):
        for wild in ((top, 1), (top, 9), (top - 1, 3)):
            got, table = run([0, wild[0], 0], [3, wild[1], 2], page, 4, 40)
            want = O.paged_tables([0], [3], np.full((1, 4), -1), free, page, 3)
            assert np.array_equal(table[:1].cpu().numpy(), want[0])
            assert np.array_equal(got.slots[:3].cpu().numpy(), want[4])
            assert got.requests[:3].tolist() == [0] * 3 and got.lengths[:3].tolist() == [1, 2, 3]
    for _ in range(20):
        for requests in (3, 300, 6000):
            past = rng.integers(0, top, requests, endpoint=True)
            past[rng.random(requests) < 0.5] //= 2 ** 28
            fresh = rng.integers(-2 ** 31, top, requests, endpoint=True)
            run(past, fresh, int(rng.integers(1, 70)), int(rng.integers(1, 9)),
                int(rng.integers(1, 9000)))


def test_select_from_several_threads():
    """Calls with tables of different widths from several host threads: their
    kernels' shared memory differs, each launch is its call's own."""
    import threading

    from mlxvs_b200 import paged

    torch = torch_()
    lib = mv._load()
    rng = np.random.default_rng(23)
    dim, n = 64, 4
    codes = on_gpu(np.sort(rng.integers(-127, 128, (50, 1, 2, dim)), 2), "int8")
    scales = torch.ones(50, 1, device="cuda")
    q = torch.randn(16, 1, dim, device="cuda").half()
    cache = paged._CACHE.pack(0, 0, 0, 0, 0, 0, 0, 0, 50, codes.data_ptr(), scales.data_ptr(), 16,
                              1, dim, 0, 1.0, 1.0)
    requests, lengths = on_gpu([0] * 16), on_gpu([40 * 16] * 16)
    calls = []
    for width in (1200, 6000):  # 38 and 192 KB for tiles of 8 tokens
        table = on_gpu(rng.integers(0, 50, (1, width)))
        want = mv.paged_select(q, codes, scales, table, lengths, 16, n, requests=requests)
        queries, _, _ = paged._queries(q, table, lengths, requests, "test")
        calls.append((table, queries, want))
    failed = []

    def work(queries, want):
        stream = torch.cuda.Stream()
        out = torch.zeros_like(want)
        stream.wait_stream(torch.cuda.current_stream())
        args = (cache, queries, n, 1, 1, out.data_ptr(), stream.cuda_stream)
        run = lib.mlxvs_paged_select_device
        for _ in range(20000):
            if run(*args):
                failed.append(lib.mlxvs_last_error())
                break
        stream.synchronize()
        if not torch.equal(out, want):
            failed.append("another result")

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=calls[i % 2][1:]) for i in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


FORMS = [("bfloat16", "bfloat16"), ("float16", "float16"), ("bfloat16", "float8_e4m3fn"),
         ("float16", "float8_e4m3fn")]


def attend_alike(kind, cache, k0, v0, scale, prompt, group=8, page=64):
    """Attention of like tokens over like requests, by the kernel of single
    tokens or the prompts'.  k0: channel 0 of the keys, where the queries are 1
    and all else is 0; v0 [keys, dim].  Returns out [.., dim] and lse [..]."""
    torch = torch_()
    heads, dim = 8, v0.shape[1]
    pages = -(-len(k0) // page)
    keys = torch.zeros(pages * page, heads, dim, device="cuda")
    values = torch.zeros_like(keys)
    keys[:len(k0), :, 0] = on_gpu(k0, "float32")[:, None]
    values[:len(k0)] = on_gpu(v0, "float32")[:, None]
    keys, values = (x.view(pages, page, heads, dim).to(dtype(cache)) for x in (keys, values))
    tokens, rows = (600, 1) if prompt else (64, 64)
    q = torch.zeros(tokens, heads * group, dim, dtype=dtype(kind), device="cuda")
    q[..., 0] = 1
    table = on_gpu(np.arange(pages)[None].repeat(rows, 0))
    more = {}
    if prompt:
        more = dict(requests=on_gpu([0] * tokens),
                    pages=on_gpu(np.arange(pages)).expand(tokens, heads, -1).contiguous())
    out, lse = mv.paged_attention(q, keys, values, table, on_gpu([len(k0)] * tokens), scale=scale,
                                  return_lse=True, **more)
    return wide(out).reshape(-1, dim), wide(lse).reshape(-1)


def exact_alike(k0, v0, scale):
    """The same for one token, in 64 bits, and its weights."""
    s = np.asarray(k0, float) * float(np.float32(scale))
    p = np.exp(s - s.max())
    with np.errstate(all="ignore"):
        return p @ v0 / p.sum(), s.max() + np.log(p.sum()), p / p.sum()


@pytest.mark.parametrize("prompt", [False, True])
@pytest.mark.parametrize("kind,cache", FORMS)
def test_weights_where_values_cancel(kind, cache, prompt):
    """200 keys of weight 1 and value 1, 400 of weight 0.5 (1 + 0.9 2^-11) and
    value -1: the sum is what a weight's rounding to 11 bits would leave.

    The weights' two terms leave 2^-17 of them at most, the tensor cores' sums
    of at most 600 / 16 steps 38 2^-23, exponentials and scores (one product)
    less than 2^-20: 2^-16 in all, and the output's own rounding."""
    weight = 0.5 * (1 + 0.9 * 2.0 ** -11)
    rng = np.random.default_rng(24)
    second = np.zeros(600)
    second[rng.permutation(600)[:400]] = 1
    v0 = np.repeat((1 - 2 * second)[:, None], 64, 1)
    scale = -np.log(weight)
    want, want_lse, _ = exact_alike(-second, v0, scale)
    out, lse = attend_alike(kind, cache, -second, v0, scale, prompt)
    assert (np.abs(out - want) <= UNIT[kind] * np.abs(want) + 2.0 ** -16).all()
    assert (np.abs(lse - want_lse) <= 2.0 ** -20 * (1 + abs(want_lse))).all()


@pytest.mark.parametrize("prompt", [False, True])
@pytest.mark.parametrize("kind,cache", FORMS)
def test_many_small_weights_behind_a_large_one(kind, cache, prompt):
    """One key of value 0 and 4,095 keys of weight 2^-25.5 behind it: the output
    is the small ones' alone.

    Float16 weights are multiples of 2^-24, 2^-7 times that of the largest one:
    off by 2^-32 at most each, the sum of 4,095 by 4,095 2^-32 times the value
    (1.1 %), beside what values that cancel are held to."""
    k0 = np.r_[0.0, np.full(4095, -1.0)]
    v0 = np.r_[0.0, np.full(4095, 256.0)][:, None].repeat(64, 1)
    scale = 25.5 * np.log(2)
    want, want_lse, _ = exact_alike(k0, v0, scale)
    out, lse = attend_alike(kind, cache, k0, v0, scale, prompt, group=1)
    tol = (UNIT[kind] + 2.0 ** -13) * want + 4095 * 2.0 ** -32 * 256
    assert (np.abs(out - want) <= tol).all()
    assert (np.abs(lse - want_lse) <= 2.0 ** -20 * (1 + abs(want_lse))).all()


@pytest.mark.parametrize("prompt", [False, True])
@pytest.mark.parametrize("kind", ["bfloat16", "float16"])
def test_infinite_values(kind, prompt):
    """A visible infinite value makes its channel infinite, both signs make it
    NaN, and other channels stay as they are."""
    rng = np.random.default_rng(25)
    k0 = rng.integers(-3, 4, 300).astype(float)
    v0 = rng.integers(-8, 9, (300, 64)).astype(float)
    plain, _ = attend_alike(kind, kind, k0, v0, 0.7, prompt)
    v0[17, 3] = np.inf
    v0[280, 4] = -np.inf
    v0[[5, 99], 5] = np.inf
    v0[[6, 100], 6] = np.inf, -np.inf
    v0[250, 7] = np.nan
    out, lse = attend_alike(kind, kind, k0, v0, 0.7, prompt)
    assert (out[:, [3, 5]] == np.inf).all() and (out[:, 4] == -np.inf).all()
    assert np.isnan(out[:, [6, 7]]).all()
    assert np.array_equal(np.delete(out, range(3, 8), 1), np.delete(plain, range(3, 8), 1))
    assert np.isfinite(lse).all()


@pytest.mark.parametrize("prompt", [False, True])
@pytest.mark.parametrize("size", [1e36, 1e-37, 2.0 ** -130])
def test_queries_of_any_size_over_an_8_bit_cache(size, prompt):
    """bfloat16 queries near the ends of their range, with a scale that makes
    their scores ordinary: as those of size 1.  Powers of two and products by
    them are exact, so only the scale's rounding is left (2^-24 of scores of at
    most 6, twice that in a weight)."""
    torch = torch_()
    rng = np.random.default_rng(26)
    page, heads, dim, length = 64, 8, 64, 300
    keys, values = make_cache(rng, 5, page, heads, dim, "float8_e4m3fn")
    tokens, rows = (600, 1) if prompt else (64, 64)
    q = torch.from_numpy(rng.integers(-3, 4, (tokens, heads, dim))).cuda().bfloat16()
    by = 2.0 ** np.floor(np.log2(size))  # exact, for subnormal ones as well
    table = on_gpu(np.arange(5)[None].repeat(rows, 0))
    more = {}
    if prompt:
        more = dict(requests=on_gpu([0] * tokens),
                    pages=on_gpu(np.arange(5)).expand(tokens, heads, -1).contiguous())
    lengths = on_gpu([length] * tokens)
    want, want_lse = mv.paged_attention(q, keys, values, table, lengths, scale=1 / 32,
                                        return_lse=True, **more)
    out, lse = mv.paged_attention((q.double() * by).bfloat16(), keys, values, table, lengths,
                                  scale=1 / 32 / by, return_lse=True, **more)
    assert np.isfinite(wide(out)).all()
    assert (np.abs(wide(lse) - wide(want_lse)) <= 2.0 ** -20 * (1 + np.abs(wide(want_lse)))).all()
    assert (np.abs(wide(out) - wide(want)) <= 2 * UNIT["bfloat16"] * np.abs(wide(want)) + 1e-5).all()

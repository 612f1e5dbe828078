"""Paged key-value cache of a language model's serving step (CUDA tensors).

    t = paged_tables(past, fresh, table, free_pages, page_size, num_tokens)
    paged_store(k, v, t.slots, keys, values, codes, scales)
    pages = paged_select(q, codes, scales, table, t.lengths, page_size, n,
                         requests=t.requests)
    out = paged_attention(q, keys, values, table, t.lengths,
                          requests=t.requests, pages=pages)

A cache is two tensors [pages, page_size, key heads, dim] (any strides with a
contiguous last dimension) of float16, bfloat16 or float8_e4m3fn, and, where
pages are to be selected, codes int8 [pages, key heads, 2, dim] and scales
float32 [pages, key heads]: bounds of each page's keys.  table int32
[requests, width] lists each request's pages in order.  Calls are queued on
the current stream (or `stream=`), allocate their outputs only, and never wait
for the GPU, so a step of fixed sizes can be captured in a CUDA graph.
"""

import collections
import struct

from . import _check, _is_torch, _load, _stream_handle, _torch

PagedTables = collections.namedtuple("PagedTables", "starts requests lengths slots used")

# mlxvs_paged_cache and mlxvs_paged_queries of include/mlxvs_c.h
_CACHE = struct.Struct("=QQqqqqqqqQQiiiiff")
_QUERIES = struct.Struct("=QqqqQqqQQii")

_types = None


def _type(t, op, name):
    global _types
    if _types is None:
        torch = _torch()
        _types = {torch.float16: 0, torch.bfloat16: 1, torch.float8_e4m3fn: 2}
    try:
        return _types[t.dtype]
    except KeyError:
        raise ValueError(f"[{op}] {name} must be float16, bfloat16 or, in a cache, "
                         f"float8_e4m3fn; got {t.dtype}.") from None


def _want(t, op, name, dtype, dim, device):
    """A contiguous CUDA tensor of the given type and number of dimensions."""
    if not (_is_torch(t) and t.dtype is dtype and t.dim() == dim and t.is_contiguous()
            and t.is_cuda):
        raise ValueError(f"[{op}] {name} must be a contiguous {dim}-D CUDA tensor of {dtype}.")
    if t.device != device:
        raise ValueError(f"[{op}] {name} must be on {device}.")


def _rows(t, op, name, dims):
    """A CUDA tensor with a contiguous last dimension."""
    if not (_is_torch(t) and t.is_cuda and t.dim() == len(dims)):
        raise ValueError(f"[{op}] {name} must be a CUDA tensor [{', '.join(dims)}].")
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"[{op}] {name} must be contiguous in its last dimension.")
    return t


def _bounds(codes, scales, op, pages, heads, dim, device):
    torch = _torch()
    _want(codes, op, "codes", torch.int8, 4, device)
    _want(scales, op, "scales", torch.float32, 2, device)
    if tuple(codes.shape) != (pages, heads, 2, dim) or tuple(scales.shape) != (pages, heads):
        raise ValueError(f"[{op}] codes must be [pages, key heads, 2, dim] and scales "
                         "[pages, key heads].")


def _cache(keys, values, codes, scales, k_scale, v_scale, op, device):
    _rows(keys, op, "keys", ("pages", "page_size", "key heads", "dim"))
    _rows(values, op, "values", ("pages", "page_size", "key heads", "dim"))
    if keys.shape != values.shape or keys.dtype != values.dtype:
        raise ValueError(f"[{op}] keys and values must have the same shape and type.")
    if keys.device != device or values.device != device:
        raise ValueError(f"[{op}] keys and values must be on {device}.")
    pages, page_size, heads, dim = keys.shape
    if codes is not None or scales is not None:
        _bounds(codes, scales, op, pages, heads, dim, device)
    ks, vs = keys.stride(), values.stride()
    return _CACHE.pack(
        keys.data_ptr(), values.data_ptr(), ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], pages,
        codes.data_ptr() if codes is not None else 0,
        scales.data_ptr() if scales is not None else 0,
        page_size, heads, dim, _type(keys, op, "keys"), k_scale, v_scale)


def _queries(q, table, lengths, requests, op):
    torch = _torch()
    _rows(q, op, "q", ("tokens", "query heads", "dim"))
    device = q.device
    _want(table, op, "table", torch.int32, 2, device)
    _want(lengths, op, "lengths", torch.int32, 1, device)
    tokens, heads, _ = q.shape
    if lengths.shape[0] != tokens:
        raise ValueError(f"[{op}] lengths must be [tokens].")
    if requests is not None:
        _want(requests, op, "requests", torch.int32, 1, device)
        if requests.shape[0] != tokens:
            raise ValueError(f"[{op}] requests must be [tokens].")
    qs = q.stride()
    return _QUERIES.pack(
        q.data_ptr(), tokens, qs[0], qs[1], table.data_ptr(), table.shape[0], table.shape[1],
        requests.data_ptr() if requests is not None else 0, lengths.data_ptr(), heads,
        _type(q, op, "q"))


class _On:
    """Makes a tensor's device current around a call; free when it already is."""

    def __init__(self, device):
        self.index = device.index

    def __enter__(self):
        cuda = _torch().cuda
        self.before = cuda.current_device()
        if self.before != self.index:
            cuda.set_device(self.index)

    def __exit__(self, *exc):
        if self.before != self.index:
            _torch().cuda.set_device(self.before)


def paged_tables(past, fresh, table, free_pages, page_size, num_tokens, *, stream=None):
    """Page tables and slot maps of one step, built on the GPU.

    past, fresh: int32 [requests], the tokens that each request holds and the
    new ones it gets.  table: int32 [requests, width]; its entries for the
    pages that a request needs beyond ceil(past / page_size) are filled in
    place from free_pages (int32, taken from the front in request order).
    num_tokens: the size of the per-token outputs, at least sum(fresh) (the
    rest is padding).

    Returns PagedTables(starts int32 [requests + 1], requests int32, lengths
    int32 and slots int64 [num_tokens], used int32 [2]): a token's request (-1
    for padding), its position + 1 (0 for padding) and its slot (page *
    page_size + row, -1 if it got none); used holds the pages taken and the
    tokens that got no slot (free_pages ended, or the table is too narrow).
    """
    op = "mlxvs::paged_tables"
    lib = _load()
    torch = _torch()
    if not (_is_torch(past) and past.is_cuda):
        raise ValueError(f"[{op}] past must be a contiguous 1-D CUDA tensor of torch.int32.")
    device = past.device
    _want(past, op, "past", torch.int32, 1, device)
    _want(fresh, op, "fresh", torch.int32, 1, device)
    _want(table, op, "table", torch.int32, 2, device)
    _want(free_pages, op, "free_pages", torch.int32, 1, device)
    requests, num_tokens = past.shape[0], int(num_tokens)
    if fresh.shape[0] != requests or table.shape[0] != requests:
        raise ValueError(f"[{op}] past, fresh and table must have one row per request.")
    if num_tokens < 0:
        raise ValueError(f"[{op}] num_tokens must be in [0, 2^31).")
    with _On(device):
        slots = torch.empty(num_tokens, dtype=torch.int64, device=device)
        ints = torch.empty(2 * num_tokens + requests + 3, dtype=torch.int32, device=device)
        rows, lengths, starts, used = ints.split((num_tokens, num_tokens, requests + 1, 2))
        at = ints.data_ptr()
        _check(lib.mlxvs_paged_tables_device(
            past.data_ptr(), fresh.data_ptr(), requests, int(page_size), free_pages.data_ptr(),
            free_pages.shape[0], table.data_ptr(), table.shape[1], num_tokens,
            at + 8 * num_tokens, at, at + 4 * num_tokens, slots.data_ptr(),
            at + 8 * num_tokens + 4 * (requests + 1), _stream_handle(stream, device)))
    return PagedTables(starts, rows, lengths, slots, used)


def paged_store(k, v, slots, keys, values, codes=None, scales=None, *, k_scale=1.0, v_scale=1.0,
                stream=None):
    """Writes the rows k, v [tokens, key heads, dim] to their slots (int64, as
    paged_tables gives them; negative ones are skipped) of the cache, times the
    float32 reciprocals of k_scale / v_scale, rounded to the cache's type,
    which is k's or float8_e4m3fn (saturating).  With codes and scales, the bounds of every
    page that got a row are renewed."""
    op = "mlxvs::paged_store"
    lib = _load()
    torch = _torch()
    _rows(k, op, "k", ("tokens", "key heads", "dim"))
    _rows(v, op, "v", ("tokens", "key heads", "dim"))
    device = k.device
    cache = _cache(keys, values, codes, scales, k_scale, v_scale, op, device)
    if k.shape != v.shape or k.dtype != v.dtype or v.device != device:
        raise ValueError(f"[{op}] k and v must have the same shape, type and device.")
    if k.shape[1:] != keys.shape[2:]:
        raise ValueError(f"[{op}] k and v must have the cache's heads and dimension.")
    _want(slots, op, "slots", torch.int64, 1, device)
    if slots.shape[0] != k.shape[0]:
        raise ValueError(f"[{op}] slots must be [tokens].")
    ks, vs = k.stride(), v.stride()
    with _On(device):
        _check(lib.mlxvs_paged_store_device(
            cache, k.data_ptr(), v.data_ptr(), _type(k, op, "k"), k.shape[0], ks[0], ks[1],
            vs[0], vs[1], slots.data_ptr(), _stream_handle(stream, device)))


def paged_select(q, codes, scales, table, lengths, page_size, n, *, requests=None, first=1,
                 last=1, stream=None):
    """The n pages that each token and key head attends to, by an 8-bit bound
    of its scores: int32 [tokens, key heads, n], positions in the request's
    row of table, ascending, -1 past the last.  The first `first` and last
    `last` pages that hold keys of the token are always among them; ties go to
    the lower page.

    q: [tokens, query heads, dim]; codes, scales: the cache's bounds; lengths:
    int32 [tokens], the keys that each token sees; requests: int32 [tokens],
    its row of the table (None: token t has row t).
    """
    op = "mlxvs::paged_select"
    lib = _load()
    torch = _torch()
    n = int(n)
    queries = _queries(q, table, lengths, requests, op)
    if not (_is_torch(codes) and codes.dim() == 4):
        raise ValueError(f"[{op}] codes must be [pages, key heads, 2, dim] and scales "
                         "[pages, key heads].")
    pages, heads, _, dim = codes.shape
    _bounds(codes, scales, op, pages, heads, q.shape[2], q.device)
    cache = _CACHE.pack(0, 0, 0, 0, 0, 0, 0, 0, pages, codes.data_ptr(), scales.data_ptr(),
                        int(page_size), heads, dim, _type(q, op, "q"), 1.0, 1.0)
    with _On(q.device):
        out = torch.empty((q.shape[0], heads, max(n, 0)), dtype=torch.int32, device=q.device)
        _check(lib.mlxvs_paged_select_device(
            cache, queries, n, int(first), int(last), out.data_ptr(),
            _stream_handle(stream, q.device)))
    return out


def paged_attention(q, keys, values, table, lengths, *, requests=None, pages=None, scale=None,
                    k_scale=1.0, v_scale=1.0, return_lse=False, stream=None):
    """Attention of each token over its request's first `lengths` keys, or over
    those of them in the pages that paged_select lists for it: softmax(scale *
    q . k) v, of q's shape and type.  scale: 1 / sqrt(dim) by default.  Query
    head i reads key head i // (query heads // key heads).  A token with no
    keys gets zeros.

    With return_lse also the logarithm of the sum of exponentials, float32
    [tokens, query heads] (-inf for a token with no keys).
    """
    op = "mlxvs::paged_attention"
    lib = _load()
    torch = _torch()
    queries = _queries(q, table, lengths, requests, op)
    device = q.device
    cache = _cache(keys, values, None, None, k_scale, v_scale, op, device)
    tokens, q_heads, dim = q.shape
    if dim != keys.shape[3]:
        raise ValueError(f"[{op}] q must have the cache's dimension.")
    n, selected = 0, None
    if pages is not None:
        _want(pages, op, "pages", torch.int32, 3, device)
        n = pages.shape[2]
        if pages.shape[0] != tokens or pages.shape[1] != keys.shape[2] or n < 1:
            raise ValueError(f"[{op}] pages must be [tokens, key heads, n].")
        selected = pages.data_ptr()
    if scale is None:
        scale = dim ** -0.5
    with _On(device):
        out = torch.empty((tokens, q_heads, dim), dtype=q.dtype, device=device)
        lse = torch.empty((tokens, q_heads), dtype=torch.float32, device=device) \
            if return_lse else None
        _check(lib.mlxvs_paged_attention_device(
            cache, queries, selected, n, scale, out.data_ptr(),
            lse.data_ptr() if return_lse else None, _stream_handle(stream, device)))
    return (out, lse) if return_lse else out

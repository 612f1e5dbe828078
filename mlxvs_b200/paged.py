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
for the GPU, so a step of fixed sizes can be captured in a CUDA graph.  They are
for inference: results carry no gradients, whatever their inputs do.
"""

import collections
import struct

from . import _check, _load

PagedTables = collections.namedtuple("PagedTables", "starts requests lengths slots used")

# mlxvs_paged_cache and mlxvs_paged_queries of include/mlxvs_c.h
_CACHE = struct.Struct("=QQqqqqqqqQQiiiiff")
_QUERIES = struct.Struct("=QqqqQqqQQii")

torch = None


def _ready():
    """The library, with torch and what is used of it: the package is imported
    without torch, which these functions need and the search does not.

    A decoding step makes these calls per layer, so their own time counts: the
    checks below read each tensor's fields once, and the stream is read without
    the Stream object that torch.cuda.current_stream builds."""
    if torch is None:
        import torch as t

        globals().update(
            Tensor=t.Tensor, float32=t.float32, int8=t.int8, int32=t.int32, int64=t.int64,
            _TYPES={t.float16: 0, t.bfloat16: 1, t.float8_e4m3fn: 2},
            _current_stream=t._C._cuda_getCurrentRawStream,
            _current_device=t.cuda.current_device, torch=t)
    return _load()


def _type(t, op, name):
    code = _TYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"[{op}] {name} must be float16, bfloat16 or, in a cache, "
                         f"float8_e4m3fn; got {t.dtype}.")
    return code


def _want(t, op, name, dtype, dim, index):
    """Checks for a contiguous tensor of the given type and number of
    dimensions on the CUDA device `index`."""
    if (isinstance(t, Tensor) and t.dtype is dtype and t.dim() == dim and t.is_contiguous()
            and t.get_device() == index):
        return
    if isinstance(t, Tensor) and t.is_cuda and t.get_device() != index:
        raise ValueError(f"[{op}] {name} must be on cuda:{index}.")
    raise ValueError(f"[{op}] {name} must be a contiguous {dim}-D CUDA tensor of {dtype}.")


def _rows(t, op, name, dims):
    """The strides of a CUDA tensor with a contiguous last dimension."""
    if not (isinstance(t, Tensor) and t.is_cuda and t.dim() == len(dims)):
        raise ValueError(f"[{op}] {name} must be a CUDA tensor [{', '.join(dims)}].")
    strides = t.stride()
    if strides[-1] != 1 and t.shape[-1] > 1:
        raise ValueError(f"[{op}] {name} must be contiguous in its last dimension.")
    return strides


def _bounds(codes, scales, op, pages, heads, dim, index):
    _want(codes, op, "codes", int8, 4, index)
    _want(scales, op, "scales", float32, 2, index)
    if codes.shape != (pages, heads, 2, dim) or scales.shape != (pages, heads):
        raise ValueError(f"[{op}] codes must be [pages, key heads, 2, dim] and scales "
                         "[pages, key heads].")


_CACHE_DIMS = ("pages", "page_size", "key heads", "dim")
_Q_DIMS = ("tokens", "query heads", "dim")
_K_DIMS = ("tokens", "key heads", "dim")


def _cache(keys, values, codes, scales, k_scale, v_scale, op, index):
    """mlxvs_paged_cache of the tensors, and their shape."""
    ks = _rows(keys, op, "keys", _CACHE_DIMS)
    vs = _rows(values, op, "values", _CACHE_DIMS)
    shape = keys.shape
    if values.shape != shape or keys.dtype is not values.dtype:
        raise ValueError(f"[{op}] keys and values must have the same shape and type.")
    if keys.get_device() != index or values.get_device() != index:
        raise ValueError(f"[{op}] keys and values must be on cuda:{index}.")
    pages, page_size, heads, dim = shape
    at_codes = at_scales = 0
    if codes is not None or scales is not None:
        _bounds(codes, scales, op, pages, heads, dim, index)
        at_codes, at_scales = codes.data_ptr(), scales.data_ptr()
    return _CACHE.pack(
        keys.data_ptr(), values.data_ptr(), ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], pages,
        at_codes, at_scales, page_size, heads, dim, _type(keys, op, "keys"), k_scale,
        v_scale), shape


def _queries(q, table, lengths, requests, op):
    """mlxvs_paged_queries of the tensors, q's shape and its device."""
    qs = _rows(q, op, "q", _Q_DIMS)
    index = q.get_device()
    _want(table, op, "table", int32, 2, index)
    _want(lengths, op, "lengths", int32, 1, index)
    shape = q.shape
    tokens = shape[0]
    if lengths.shape[0] != tokens:
        raise ValueError(f"[{op}] lengths must be [tokens].")
    at_requests = 0
    if requests is not None:
        _want(requests, op, "requests", int32, 1, index)
        if requests.shape[0] != tokens:
            raise ValueError(f"[{op}] requests must be [tokens].")
        at_requests = requests.data_ptr()
    rows, width = table.shape
    return _QUERIES.pack(
        q.data_ptr(), tokens, qs[0], qs[1], table.data_ptr(), rows, width, at_requests,
        lengths.data_ptr(), shape[1], _type(q, op, "q")), shape, index


def _whole(x, op, what, low=-2**31, high=2**31):
    """A whole number that the C entries take in 32 bits (their range checks
    would see what is left of a larger one)."""
    x = int(x)
    if not low <= x < high:
        raise ValueError(f"[{op}] {what}")
    return x


_PAGE_SIZE = "page_size must be in [1, 1024]."
_N = "n must be in [1, 256]."
_ENDS = "first and last must be at least 0 and together at most n."
_TOKENS = "num_tokens must be in [0, 2^31)."


def _stream(stream, index):
    """A context in which `stream` (a torch stream or a cudaStream_t) is the
    current one, so that outputs are allocated in its order as well."""
    if isinstance(stream, int):
        stream = torch.cuda.ExternalStream(stream, device=torch.device("cuda", index))
    return torch.cuda.stream(stream)


def _call(function, args, index):
    """A C entry with the stream as its last argument, on device `index`."""
    handle = _current_stream(index)
    if _current_device() == index:
        rc = function(*args, handle)
    else:
        with torch.cuda.device(index):
            rc = function(*args, handle)
    if rc:
        _check(rc)


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
    lib = _ready()
    page_size = _whole(page_size, op, _PAGE_SIZE)
    num_tokens = _whole(num_tokens, op, _TOKENS, 0)
    if not (isinstance(past, Tensor) and past.is_cuda):
        raise ValueError(f"[{op}] past must be a contiguous 1-D CUDA tensor of torch.int32.")
    index = past.get_device()
    if stream is not None:
        with _stream(stream, index):
            return paged_tables(past, fresh, table, free_pages, page_size, num_tokens)
    _want(past, op, "past", int32, 1, index)
    _want(fresh, op, "fresh", int32, 1, index)
    _want(table, op, "table", int32, 2, index)
    _want(free_pages, op, "free_pages", int32, 1, index)
    requests = past.shape[0]
    rows, width = table.shape
    if fresh.shape[0] != requests or rows != requests:
        raise ValueError(f"[{op}] past, fresh and table must have one row per request.")
    slots = past.new_empty(num_tokens, dtype=int64)
    ints = past.new_empty(2 * num_tokens + requests + 3)
    at = ints.data_ptr()
    starts = at + 8 * num_tokens
    _call(lib.mlxvs_paged_tables_device,
          (past.data_ptr(), fresh.data_ptr(), requests, page_size, free_pages.data_ptr(),
           free_pages.shape[0], table.data_ptr(), width, num_tokens, starts, at,
           at + 4 * num_tokens, slots.data_ptr(), starts + 4 * (requests + 1)), index)
    of, lengths, starts, used = torch.split_with_sizes(
        ints, (num_tokens, num_tokens, requests + 1, 2))
    return PagedTables(starts, of, lengths, slots, used)


def paged_store(k, v, slots, keys, values, codes=None, scales=None, *, k_scale=1.0, v_scale=1.0,
                stream=None):
    """Writes the rows k, v [tokens, key heads, dim] to their slots (int64, as
    paged_tables gives them; those outside the cache are skipped), times the
    float32 reciprocals of k_scale / v_scale, rounded to the cache's type,
    which is k's or float8_e4m3fn (saturating).  With codes and scales, the bounds of every
    page that got a row are renewed, over its rows up to the last new one.

    Slots must differ, and a page's new rows be tokens in a row, one row on for
    each token; any of them may be skipped, which leaves its row as it was."""
    op = "mlxvs::paged_store"
    lib = _ready()
    ks = _rows(k, op, "k", _K_DIMS)
    vs = _rows(v, op, "v", _K_DIMS)
    index = k.get_device()
    if stream is not None:
        with _stream(stream, index):
            return paged_store(k, v, slots, keys, values, codes, scales, k_scale=k_scale,
                               v_scale=v_scale)
    cache, shape = _cache(keys, values, codes, scales, k_scale, v_scale, op, index)
    if k.shape != v.shape or k.dtype is not v.dtype or v.get_device() != index:
        raise ValueError(f"[{op}] k and v must have the same shape, type and device.")
    if k.shape[1:] != shape[2:]:
        raise ValueError(f"[{op}] k and v must have the cache's heads and dimension.")
    tokens = k.shape[0]
    _want(slots, op, "slots", int64, 1, index)
    if slots.shape[0] != tokens:
        raise ValueError(f"[{op}] slots must be [tokens].")
    _call(lib.mlxvs_paged_store_device,
          (cache, k.data_ptr(), v.data_ptr(), _type(k, op, "k"), tokens, ks[0], ks[1], vs[0],
           vs[1], slots.data_ptr()), index)


def paged_select(q, codes, scales, table, lengths, page_size, n, *, requests=None, first=1,
                 last=1, stream=None):
    """The n pages that each token and key head attends to, by an 8-bit estimate
    of the bound of its scores: int32 [tokens, key heads, n], positions in the request's
    row of table, ascending, -1 past the last.  The first `first` and last
    `last` pages that hold keys of the token are always among them; ties go to
    the lower page.

    q: [tokens, query heads, dim]; codes, scales: the cache's bounds; lengths:
    int32 [tokens], the keys that each token sees; requests: int32 [tokens],
    its row of the table (None: token t has row t).
    """
    op = "mlxvs::paged_select"
    lib = _ready()
    n = _whole(n, op, _N, 1, 257)
    page_size = _whole(page_size, op, _PAGE_SIZE)
    first, last = _whole(first, op, _ENDS), _whole(last, op, _ENDS)
    queries, shape, index = _queries(q, table, lengths, requests, op)
    if stream is not None:
        with _stream(stream, index):
            return paged_select(q, codes, scales, table, lengths, page_size, n,
                                requests=requests, first=first, last=last)
    if not (isinstance(codes, Tensor) and codes.dim() == 4):
        raise ValueError(f"[{op}] codes must be [pages, key heads, 2, dim] and scales "
                         "[pages, key heads].")
    pages, heads = codes.shape[:2]
    _bounds(codes, scales, op, pages, heads, shape[2], index)
    cache = _CACHE.pack(0, 0, 0, 0, 0, 0, 0, 0, pages, codes.data_ptr(), scales.data_ptr(),
                        page_size, heads, shape[2], _type(q, op, "q"), 1.0, 1.0)
    out = table.new_empty((shape[0], heads, n))
    _call(lib.mlxvs_paged_select_device,
          (cache, queries, n, first, last, out.data_ptr()), index)
    return out


def paged_attention(q, keys, values, table, lengths, *, requests=None, pages=None, scale=None,
                    k_scale=1.0, v_scale=1.0, return_lse=False, stream=None):
    """Attention of each token over its request's first `lengths` keys, or over
    those of them in the pages that paged_select lists for it (a page at most
    once for a token and key head): softmax(scale * q . k) v, of q's shape and
    type.  scale: 1 / sqrt(dim) by default.  Query
    head i reads key head i // (query heads // key heads).  A token with no
    keys gets zeros.

    With return_lse also the logarithm of the sum of exponentials, float32
    [tokens, query heads] (-inf for a token with no keys).
    """
    op = "mlxvs::paged_attention"
    lib = _ready()
    queries, shape, index = _queries(q, table, lengths, requests, op)
    if stream is not None:
        with _stream(stream, index):
            return paged_attention(q, keys, values, table, lengths, requests=requests,
                                   pages=pages, scale=scale, k_scale=k_scale, v_scale=v_scale,
                                   return_lse=return_lse)
    cache, kv = _cache(keys, values, None, None, k_scale, v_scale, op, index)
    tokens, q_heads, dim = shape
    if dim != kv[3]:
        raise ValueError(f"[{op}] q must have the cache's dimension.")
    n = at_pages = 0
    if pages is not None:
        _want(pages, op, "pages", int32, 3, index)
        of, heads, n = pages.shape
        if of != tokens or heads != kv[2] or n < 1:
            raise ValueError(f"[{op}] pages must be [tokens, key heads, n].")
        at_pages = pages.data_ptr()
    if scale is None:
        scale = dim ** -0.5
    out = torch.empty_like(q) if q.is_contiguous() else q.new_empty(shape)
    lse = q.new_empty((tokens, q_heads), dtype=float32) if return_lse else None
    _call(lib.mlxvs_paged_attention_device,
          (cache, queries, at_pages, n, scale, out.data_ptr(),
           lse.data_ptr() if return_lse else None), index)
    return (out, lse) if return_lse else out

"""A paged key-value cache for token generation: its upkeep and the attention over it, executed by libmq.so on
the current HIP stream. (No counterpart in the reference, whose attention runs in the programs that call it.)

The cache of one layer is K and V [pages, kv_heads, page_size, head_dim] in bf16, fp16 or, with fp32 scales
[pages, kv_heads, page_size], int8 (any order of the dimensions in memory, head_dim contiguous, K and V
alike). Token j of sequence b lies in slot j % page_size of page page_table[b, j // page_size]; page_size is a power of
two. page_table (int32 [seqs, width], -1: no page), kv_lens (int32 [seqs], tokens held, the new ones among
them), refs (int32 [pages], sequences that hold a page) and cu_q (int32 [seqs + 1], where each sequence's new
tokens begin; None: one new token each) stay on the device: no call waits for it or reads from it.

    cache = ck.PagedKVCache(layers=2, pages=512, kv_heads=8, head_dim=128, seqs=16, max_tokens=4096)
    cache.grow(range(16), [1] * 16)             # room for a token each
    cache.write(layer, k, v)                    # k, v [16, 8, 128]
    y = cache.attend(layer, q)                  # q [16, 32, 128]

Every call raises ValueError for tensors whose shapes, types, strides or devices do not fit. What only the
device can see is bounded there: a table entry that is no page of the cache holds nothing, and a fork or
growth that cannot be done whole changes nothing and says so in `status`.
"""
from __future__ import annotations

import threading

import torch

from . import _lib
from .ops import _scratch

CACHE_TYPES = (torch.bfloat16, torch.float16, torch.int8)
_CODE = {torch.bfloat16: _lib.DT_BF16, torch.float16: _lib.DT_F16, torch.int8: _lib.DT_I8}
_ATTN_WS: dict = {}


class _Counters(threading.local):
    def __init__(self):
        self.by_stream: dict = {}   # (device index, stream) -> zeros


_COUNTERS = _Counters()


def _counters(n: int, device, stream: int) -> torch.Tensor:
    """Zeros that every call leaves as zeros: kept per thread, device and stream like the workspaces, whose calls
    run in order; a captured call has its own, cleared by the graph."""
    if torch.cuda.is_current_stream_capturing():
        return torch.zeros(n, dtype=torch.int32, device=device)
    kept, key = _COUNTERS.by_stream, (device.index, stream)
    buf = kept.get(key)
    if buf is None or buf.numel() < n:
        buf = kept[key] = torch.zeros(max(n, 4096), dtype=torch.int32, device=device)
    return buf


def _device_of(t: torch.Tensor, what: str):
    if not t.is_cuda:
        raise ValueError(f"kitchen_amd ops run on the GPU: {what} must be a device tensor")
    return t.device


def _rows(x: torch.Tensor, what: str) -> torch.Tensor:
    """[T, heads, D] with rows that start at multiples of 16 bytes (copied where they do not)."""
    if x.dim() != 3:
        raise ValueError(f"{what} must be [tokens, heads, head_dim], got {list(x.shape)}")
    s0, s1, s2 = x.stride()
    if s2 != 1 or s0 % 8 or s1 % 8 or x.data_ptr() % 16:
        return x.clone(memory_format=torch.contiguous_format)
    return x


def _cache_args(k, v, ks, vs, like: torch.Tensor, heads: int | None):
    """(pages, kv_heads, page_size, the library's arguments of the caches): checks a layer's caches against the tokens."""
    if k.dim() != 4 or k.shape != v.shape or k.stride() != v.stride():
        raise ValueError(f"the caches must be [pages, kv_heads, page_size, head_dim] and alike, got {list(k.shape)} and "
                         f"{list(v.shape)} (strides {k.stride()}, {v.stride()})")
    dev, dt = like.device, k.dtype
    if dt not in CACHE_TYPES or v.dtype != dt or (dt != torch.int8 and dt != like.dtype):
        raise ValueError(f"the caches must both be {like.dtype} or int8, got {dt} and {v.dtype}")
    pages, h, page, d = k.shape
    if like.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"the tokens must be bfloat16 or float16, got {like.dtype}")
    if d != like.shape[2] or (heads is not None and h != heads):
        raise ValueError(f"caches of {h} heads of {d} do not take rows {list(like.shape)}")
    if k.device != dev or v.device != dev:
        raise ValueError(f"the caches are on {k.device}, the tokens on {dev}")
    c0, c1, c2, c3 = k.stride()
    if c3 != 1 and d > 1:
        raise ValueError("head_dim must be contiguous in the caches")
    if dt == torch.int8:
        if ks is None or vs is None:
            raise ValueError("an int8 cache needs k_scale and v_scale")
        if ks.shape != k.shape[:3] or vs.shape != ks.shape or ks.stride() != vs.stride() or ks.dtype != torch.float32 \
                or vs.dtype != torch.float32 or ks.device != dev or vs.device != dev:
            raise ValueError(f"k_scale and v_scale must be float32 {list(k.shape[:3])} on {dev} with equal strides")
        s0, s1, s2 = ks.stride()
        sp = (ks.data_ptr(), vs.data_ptr(), s0, s1, s2)
    else:
        if ks is not None or vs is not None:
            raise ValueError("scales are for int8 caches")
        sp = (None, None, 0, 0, 0)
    return pages, h, page, (k.data_ptr(), v.data_ptr(), _CODE[dt], c0, c1, c2, *sp, pages, page)


def _apart(page_table: torch.Tensor) -> torch.Tensor:
    """A table that is only read, its rows behind each other (copied where they overlap, as an expanded one's do)."""
    if page_table.dim() == 2 and page_table.shape[0] > 1 and page_table.stride(0) < page_table.shape[1]:
        return page_table.contiguous()
    return page_table


def _table_args(page_table, kv_lens, cu_q, tokens: int, dev):
    """The library's arguments of the tables: (page_table, ld, sequences, width, lens, cu_q)."""
    if page_table.dim() != 2 or page_table.dtype != torch.int32 or page_table.device != dev:
        raise ValueError(f"page_table must be int32 [sequences, width] on {dev}")
    b, width = page_table.shape
    ld, unit = page_table.stride()
    if unit != 1 and width > 1:
        raise ValueError("page_table needs contiguous rows")
    if kv_lens.dtype != torch.int32 or kv_lens.dim() != 1 or kv_lens.shape[0] != b or kv_lens.device != dev \
            or not kv_lens.is_contiguous():
        raise ValueError(f"kv_lens must be contiguous int32 [{b}] on {dev}")
    cu = None
    if cu_q is None:
        if tokens != b:
            raise ValueError(f"{tokens} tokens for {b} sequences: without cu_q every sequence has one")
    else:
        if cu_q.dtype != torch.int32 or cu_q.dim() != 1 or cu_q.shape[0] != b + 1 or cu_q.device != dev \
                or not cu_q.is_contiguous():
            raise ValueError(f"cu_q must be contiguous int32 [{b + 1}] on {dev}")
        cu = cu_q.data_ptr()
    return page_table.data_ptr(), max(ld, width), b, width, kv_lens.data_ptr(), cu


def kv_write(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
             kv_lens: torch.Tensor, cu_q: torch.Tensor | None = None, k_scale: torch.Tensor | None = None,
             v_scale: torch.Tensor | None = None) -> None:
    """New tokens' keys and values k, v [tokens, kv_heads, head_dim] into their sequences' pages: new token i
    of the n of a sequence goes to position kv_lens - n + i (a position below 0 or without a page is dropped).
    An int8 cache gets codes rne(x / s) with s = max(absmax / 127, 1e-10) per token and head."""
    dev = _device_of(k, "k")
    if k.shape != v.shape or k.dtype != v.dtype or v.device != dev:
        raise ValueError(f"k and v must be alike, got {list(k.shape)} {k.dtype} and {list(v.shape)} {v.dtype}")
    k, v = _rows(k, "k"), _rows(v, "v")
    t, h, d = k.shape
    pages, _, _, cache = _cache_args(k_cache, v_cache, k_scale, v_scale, k, h)
    page_table = _apart(page_table)
    tables = _table_args(page_table, kv_lens, cu_q, t, dev)
    _lib.call("mq_kv_write", k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1),
              _CODE[k.dtype], t, h, d, *cache, *tables, _lib.stream_of_device(dev))


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                    kv_lens: torch.Tensor, cu_q: torch.Tensor | None = None, scale: float | None = None,
                    window: int | None = None, sinks: int = 0, k_scale: torch.Tensor | None = None,
                    v_scale: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of new tokens q [tokens, heads, head_dim] over their sequences' pages, causal: the query at
    position p (new token i of n: kv_lens - n + i) sees tokens j <= p, with `window` only the last `window` of
    them (its own among them) and the first `sinks`. heads is a multiple of kv_heads (query head h reads cache
    head h // (heads // kv_heads)). scale: of the scores, head_dim ** -0.5 by default. A query that sees nothing
    gets zeros. cu_q None: one new token per sequence (generation), else ragged prompt chunks.
    Returns out [tokens, heads, head_dim] in q's type."""
    dev = _device_of(q, "q")
    q = _rows(q, "q")
    t, heads, d = q.shape
    pages, h, _, cache = _cache_args(k_cache, v_cache, k_scale, v_scale, q, None)
    if h == 0 or heads % h:
        raise ValueError(f"{heads} query heads for {h} cache heads: expected a multiple")
    page_table = _apart(page_table)
    tables = _table_args(page_table, kv_lens, cu_q, t, dev)
    if window is not None and window < 1 or sinks < 0:
        raise ValueError(f"window must be at least 1 (None: no window) and sinks at least 0, got {window} and {sinks}")
    if out is None:
        out = torch.empty((t, heads, d), dtype=q.dtype, device=dev)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != dev or out.stride(2) != 1 \
            or out.stride(0) % 8 or out.stride(1) % 8 or out.data_ptr() % 16:
        raise ValueError(f"out must be {q.dtype} {list(q.shape)} on {dev} with rows at multiples of 16 bytes")
    stream = _lib.stream_of_device(dev)
    key = (dev.index, t, heads, h, d, tables[2], cu_q is None)
    sizes = _ATTN_WS.get(key)
    if sizes is None:
        lib, b, ragged = _lib.load(), tables[2], int(cu_q is not None)
        with torch.cuda.device(dev):
            sizes = (int(lib.mq_paged_attention_workspace_bytes(t, heads, h, d, b, ragged)),
                     int(lib.mq_paged_attention_counters(t, heads, h, b, ragged)))
        if len(_ATTN_WS) > 4096:   # ragged batches come in any size: the sizes are only remembered, not needed
            _ATTN_WS.clear()
        _ATTN_WS[key] = sizes
    nbytes, ncount = sizes
    work = _scratch(nbytes, dev, stream) if nbytes else None
    count = _counters(ncount, dev, stream) if ncount else None
    _lib.call("mq_paged_attention", q.data_ptr(), q.stride(0), q.stride(1), _CODE[q.dtype], t, heads, h, d, *cache,
              *tables, d ** -0.5 if scale is None else float(scale), window or 0, int(sinks), out.data_ptr(),
              out.stride(0), out.stride(1), None if work is None else work.data_ptr(), nbytes,
              None if count is None else count.data_ptr(), stream)
    return out


# --------------------------------------------------------------------------- pages

def _index(x, dev, what: str) -> torch.Tensor:
    """Sequence numbers or counts as contiguous int32 on the device."""
    if isinstance(x, torch.Tensor):
        if x.dim() != 1:
            raise ValueError(f"{what} must be one-dimensional, got {list(x.shape)}")
        return x.to(device=dev, dtype=torch.int32).contiguous()
    return torch.tensor(list(x), dtype=torch.int32, device=dev)


def _tables(page_table, lens, refs):
    dev = _device_of(page_table, "page_table")
    if page_table.dim() != 2 or page_table.dtype != torch.int32 or (page_table.stride(1) != 1 and page_table.shape[1] > 1):
        raise ValueError("page_table must be int32 [sequences, width] with contiguous rows")
    rows, width = page_table.shape
    if rows > 1 and page_table.stride(0) < width:
        raise ValueError(f"the rows of page_table must not overlap (strides {page_table.stride()})")
    for t, n, what in ((lens, rows, "lens"), (refs, None, "refs")):
        if t is not None and (t.dtype != torch.int32 or t.dim() != 1 or t.device != dev or not t.is_contiguous()
                              or (n is not None and t.shape[0] != n)):
            raise ValueError(f"{what} must be contiguous int32 [{'pages' if n is None else n}] on {dev}")
    return dev, page_table.data_ptr(), max(page_table.stride(0), width), rows, width


def _status_ptr(status, dev):
    if status is None:
        return None
    if status.dtype != torch.int32 or status.numel() < 1 or status.device != dev:
        raise ValueError(f"status must be an int32 tensor on {dev}")
    return status.data_ptr()


def _layers(k, v, ks, vs, pages: int, dev):
    """(page_size, the library's arguments of whole caches [layers, pages, kv_heads, page_size, head_dim], or one
    layer without the first dimension): every page one block of memory."""
    def block(t, dims, what):
        if t.dim() == dims - 1:
            t = t.unsqueeze(0)
        if t.dim() != dims or t.shape[1] != pages:
            raise ValueError(f"{what} must be [layers, {pages}, kv_heads, page_size{', head_dim' if dims == 5 else ''}], "
                             f"got {list(t.shape)}")
        size = 1
        for st, n in sorted((st, n) for st, n in zip(t.stride()[2:], t.shape[2:]) if n != 1):
            if st != size:
                raise ValueError(f"{what}: a page must be one block of memory (strides {t.stride()})")
            size *= n
        e = t.element_size()
        return t, (t.stride(0) * e, t.stride(1) * e, size * e)

    if k.shape != v.shape or k.stride() != v.stride() or k.dtype != v.dtype or k.device != v.device:
        raise ValueError("k and v must be alike")
    if any(t is not None and t.device != dev for t in (k, ks, vs)):
        raise ValueError(f"the caches and their scales must be on {dev}, like page_table")
    k5, args = block(k, 5, "the caches")
    sargs = (None, None, 0, 0, 0)
    if (ks is None) != (vs is None) or (k.dtype == torch.int8) != (ks is not None):
        raise ValueError("int8 caches take k_scale and v_scale, others none")
    if ks is not None:
        if ks.shape != vs.shape or ks.stride() != vs.stride() or ks.dtype != torch.float32 or vs.dtype != torch.float32:
            raise ValueError("k_scale and v_scale must be float32 and alike")
        s4, s = block(ks, 4, "the scales")
        if s4.shape != k5.shape[:4]:
            raise ValueError(f"the scales must be {list(k5.shape[:4])}, got {list(s4.shape)}")
        sargs = (ks.data_ptr(), vs.data_ptr(), *s)
    return k5.shape[3], (k.data_ptr(), v.data_ptr(), k5.shape[0], *args, *sargs)


def _kv_scratch(pages: int, n: int, dev, stream: int):
    nbytes = 4 * (2 * pages + 3 * n + 4)   # mq_kv_workspace_bytes
    return _scratch(nbytes, dev, stream), nbytes


def kv_fork(k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor, src, dst,
            k_scale=None, v_scale=None, status: torch.Tensor | None = None) -> None:
    """Sequences dst (empty) become copies of src, pairwise: full pages are shared (refs), a partly filled last
    page is copied, in every layer, to the lowest free page. k, v: the whole cache [layers, pages, kv_heads,
    page_size, head_dim] (or one layer of it). status (int32 on the device): 0 done, > 0 pages missing, -1 a row out
    of range, given twice or not empty, or a src without a page that its length asks for; nothing has changed unless it
    is 0."""
    dev, *tab = _tables(page_table, lens, refs)
    pages = refs.shape[0]
    page, cache = _layers(k, v, k_scale, v_scale, pages, dev)
    s, d = _index(src, dev, "src"), _index(dst, dev, "dst")
    n = s.shape[0]
    if d.shape[0] != n:
        raise ValueError(f"{n} sequences to fork into {d.shape[0]}")
    stream = _lib.stream_of_device(dev)
    work, nbytes = _kv_scratch(pages, n, dev, stream)
    _lib.call("mq_kv_fork", *cache, *tab, lens.data_ptr(), refs.data_ptr(), pages, page, s.data_ptr(), d.data_ptr(), n,
              _status_ptr(status, dev), work.data_ptr(), nbytes, stream)


def kv_grow(page_table: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor, seqs, counts, page_size: int,
            status: torch.Tensor | None = None) -> None:
    """counts[i] tokens more for sequence seqs[i]: lens and the lowest free pages that they need (kv_write fills
    them). status as for kv_fork."""
    dev, *tab = _tables(page_table, lens, refs)
    s, c = _index(seqs, dev, "seqs"), _index(counts, dev, "counts")
    n, pages = s.shape[0], refs.shape[0]
    if c.shape[0] != n:
        raise ValueError(f"{c.shape[0]} counts for {n} sequences")
    stream = _lib.stream_of_device(dev)
    work, nbytes = _kv_scratch(pages, n, dev, stream)
    _lib.call("mq_kv_grow", *tab, lens.data_ptr(), refs.data_ptr(), pages, int(page_size), s.data_ptr(), c.data_ptr(), n,
              _status_ptr(status, dev), work.data_ptr(), nbytes, stream)


def kv_free(page_table: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor, seqs) -> None:
    """Sequences seqs give their pages back and are empty afterwards."""
    dev, *tab = _tables(page_table, lens, refs)
    s = _index(seqs, dev, "seqs")
    _lib.call("mq_kv_free", *tab, lens.data_ptr(), refs.data_ptr(), refs.shape[0], s.data_ptr(), s.shape[0],
              _lib.stream_of_device(dev))


def kv_compact(k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor, refs: torch.Tensor, k_scale=None,
               v_scale=None) -> torch.Tensor:
    """The pages held move together: n of them are pages 0 .. n - 1 afterwards, in page_table too, with the
    fewest copies (held pages at n and above go to the free ones below n, both in ascending order).
    Returns n, int32 [1] on the device."""
    dev, *tab = _tables(page_table, None, refs)
    pages = refs.shape[0]
    _, cache = _layers(k, v, k_scale, v_scale, pages, dev)
    live = torch.empty(1, dtype=torch.int32, device=dev)
    stream = _lib.stream_of_device(dev)
    work, nbytes = _kv_scratch(pages, 0, dev, stream)
    _lib.call("mq_kv_compact", *cache, *tab, refs.data_ptr(), pages, live.data_ptr(), work.data_ptr(), nbytes, stream)
    return live


class PagedKVCache:
    """The caches of all layers with their tables, and the calls above on them.

    layers, pages, kv_heads, head_dim, page_size: shape of the cache; seqs: sequences held at once; max_tokens: the
    longest (width of the page table); dtype: bf16 or fp16, the type of the tokens; int8: hold the cache in
    8 bits. Tables and counts (page_table, lens, refs, status) are device tensors."""

    def __init__(self, layers: int, pages: int, kv_heads: int, head_dim: int, page_size: int = 16, seqs: int = 1,
                 max_tokens: int = 4096, dtype=torch.bfloat16, int8: bool = False, device="cuda"):
        if page_size < 1 or page_size & (page_size - 1):
            raise ValueError(f"page_size must be a power of two, got {page_size}")
        shape = (layers, pages, kv_heads, page_size, head_dim)
        self.page_size, self.dtype = page_size, dtype
        self.k, self.v = (torch.zeros(shape, dtype=torch.int8 if int8 else dtype, device=device) for _ in range(2))
        self.k_scale, self.v_scale = \
            (torch.zeros(shape[:4], dtype=torch.float32, device=device) if int8 else None for _ in range(2))
        width = -(-max_tokens // page_size)
        self.page_table = torch.full((seqs, width), -1, dtype=torch.int32, device=device)
        self.lens = torch.zeros(seqs, dtype=torch.int32, device=device)
        self.refs = torch.zeros(pages, dtype=torch.int32, device=device)
        self.status = torch.zeros(1, dtype=torch.int32, device=device)

    def _layer(self, layer: int):
        return (self.k[layer], self.v[layer], None if self.k_scale is None else self.k_scale[layer],
                None if self.v_scale is None else self.v_scale[layer])

    def grow(self, seqs, counts) -> None:
        kv_grow(self.page_table, self.lens, self.refs, seqs, counts, self.page_size, self.status)

    def fork(self, src, dst) -> None:
        kv_fork(self.k, self.v, self.page_table, self.lens, self.refs, src, dst, self.k_scale, self.v_scale, self.status)

    def free(self, seqs) -> None:
        kv_free(self.page_table, self.lens, self.refs, seqs)

    def compact(self) -> torch.Tensor:
        return kv_compact(self.k, self.v, self.page_table, self.refs, self.k_scale, self.v_scale)

    def check(self) -> None:
        """Waits for the device; raises if the last grow or fork could not be done."""
        code = int(self.status.item())
        if code > 0:
            raise _lib.MQError(f"the cache is {code} pages short")
        if code < 0:
            raise ValueError("a sequence is out of range, given twice, not empty, without a page that it should have, or too "
                             "long for its page table")

    def write(self, layer: int, k: torch.Tensor, v: torch.Tensor, cu_q: torch.Tensor | None = None,
              lens: torch.Tensor | None = None) -> None:
        """lens: other lengths than the cache's own, such as 0 for a sequence that gets no token in this call."""
        kc, vc, ks, vs = self._layer(layer)
        kv_write(k, v, kc, vc, self.page_table, self.lens if lens is None else lens, cu_q, ks, vs)

    def attend(self, layer: int, q: torch.Tensor, cu_q: torch.Tensor | None = None, scale: float | None = None,
               window: int | None = None, sinks: int = 0, out: torch.Tensor | None = None,
               lens: torch.Tensor | None = None) -> torch.Tensor:
        kc, vc, ks, vs = self._layer(layer)
        return paged_attention(q, kc, vc, self.page_table, self.lens if lens is None else lens, cu_q, scale, window, sinks,
                               ks, vs, out)

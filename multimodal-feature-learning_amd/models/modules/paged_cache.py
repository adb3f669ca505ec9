"""Paged key / value cache of the caption decoders as HIP kernels (csrc/paged_attention.hip,
csrc/paged_cache.hip, include/paged_cache.h): attention of a chunk of new tokens over the cache, and the page
pool's forks, cuts, growth and compaction.

The reference has no cache: it re-runs the decoder over the whole prefix for every word
(models/deformable/unimodal_deformable_dvc.py:318-354).  ``CaptionKVCache`` (layers.py) keeps dense rows for the
greedy loop; here rows share the pages of a common beginning, so beams fork without copying what they share, a
prompt enters as one chunk, and rows of very different lengths take the memory that they use.

Everything is decided on the device and on the current stream: no call waits for the host, and all may be captured.
Inference only, no CPU implementation.
"""
import struct

import torch

from ... import _native

__all__ = ["paged_attention", "pages_update", "pages_compact", "pages_copy", "PagedKVCache"]

_DTYPES = {torch.float32: 0, torch.bfloat16: 2, torch.float16: 3}
_ARGS = struct.Struct("=11Q22qd")  # mfl_paged_attention_args


_NO_STRIDES = (0, 0, 0, 0)


def _error(who):
    raise RuntimeError(f"{who}: " + _native.load_library().mfl_paged_last_error().decode(errors="replace"))


def _i32(who, name, t, shape):
    if t.dtype != torch.int32:
        raise TypeError(f"{who}: {name} must be int32, got {t.dtype}")
    if tuple(t.shape) != shape:
        raise ValueError(f"{who}: {name} must be {shape}, got {tuple(t.shape)}")
    return t if t.is_contiguous() else t.contiguous()


def _rows16(t):
    """(t, its strides) with a contiguous last dimension, 16-byte aligned rows and start (copied only if it has not)."""
    st = t.stride()
    mask = 16 // t.element_size() - 1
    if t.data_ptr() % 16 == 0 and st[-1] == 1:
        if not (st[-2] | st[-3] | st[0]) & mask:
            return t, st
        st = tuple(0 if n == 1 else x for x, n in zip(st, t.shape))  # (a dimension of one may have any stride)
        if not (st[-2] | st[-3] | st[0]) & mask:
            return t, st
    t = t.clone(memory_format=torch.contiguous_format)
    return t, t.stride()


def paged_attention(q, k_pages, v_pages, table, kv_lens, *, k=None, v=None, starts=None, offsets=None, max_rows=None,
                    max_kv=None, scale=None, causal=True, out=None):
    """Attention of new tokens over a paged cache; a single new token a sequence is the decode step.

    q: (n, rows, heads, dim), or packed (total, heads, dim) with ``offsets`` (n + 1) int32: sequence s has the
    rows offsets[s] .. offsets[s + 1].  k_pages, v_pages: (pages, kv_heads, page_size, dim), page_size a power of two up to
    1024; query head h reads key head h // (heads // kv_heads).  table (n, width) int32: key j of sequence s is row
    j % page_size of page table[s, j // page_size].  kv_lens (n) int32: cached tokens, the chunk's own included.
    ``starts`` (n) int32: the position of each sequence's first row (default: its rows end the cache).

    Row i at position p = starts + i sees the keys j < kv_lens with j <= p (``causal``) whose page number is in
    range; a row that sees nothing is 0.  ``k`` / ``v`` (q's layout with kv_heads): the chunk's own keys and values —
    row i's are written to the pages at p, where p is in [0, kv_lens), and attended.  The positions written must
    lie in pages that no other sequence reads (``pages_update`` sees to it).

    ``max_rows``: the largest number of rows of a packed sequence (rows beyond it are neither computed nor written: what
    a new tensor holds there is undefined; default: total).  ``max_kv`` guides the launch only (default: what the table
    holds).  ``scale``: dim ** -0.5.
    Returns ``out``, q's shape and type, contiguous; packed rows before the first sequence and behind the last are
    0 in a new tensor and stay as they were in a given one.  float32, bfloat16 and float16; dim up to 128, a multiple of
    16 bytes; float32 statistics.  No gradients.
    """
    who = "paged_attention"
    dt = q.dtype
    tag = _DTYPES.get(dt)
    if tag is None:
        raise TypeError(f"{who}: unsupported dtype {dt}")
    packed = offsets is not None
    shape = q.shape
    if len(shape) != (3 if packed else 4):
        raise ValueError(f"{who}: q must be {'(total, heads, dim)' if packed else '(n, rows, heads, dim)'}; got "
                         f"{tuple(shape)}")
    if k_pages.dim() != 4 or k_pages.shape != v_pages.shape:
        raise ValueError(f"{who}: k_pages {tuple(k_pages.shape)} and v_pages {tuple(v_pages.shape)} must be (pages, "
                         "kv_heads, page_size, dim)")
    if table.dim() != 2:
        raise ValueError(f"{who}: table must be (n, width); got {tuple(table.shape)}")
    n, width = table.shape
    pages, kvh, ps, d = k_pages.shape
    heads = shape[-2]
    if shape[-1] != d or kvh < 1 or heads < 1 or heads % kvh:
        raise ValueError(f"{who}: q heads x dim {tuple(shape[-2:])} do not fit pages {tuple(k_pages.shape)}")
    if packed:
        total = shape[0]
        rows = total if max_rows is None else min(int(max_rows), total)
        if rows < 0:
            raise ValueError(f"{who}: max_rows {max_rows}")
        offsets = _i32(who, "offsets", offsets, (n + 1,))
    else:
        total, rows = 0, shape[1]
        if shape[0] != n:
            raise ValueError(f"{who}: q has {shape[0]} sequences, table {n}")
    if (k is None) != (v is None):
        raise ValueError(f"{who}: k and v come together")
    if k_pages.dtype != dt or v_pages.dtype != dt or k is not None and (k.dtype != dt or v.dtype != dt):
        raise TypeError(f"{who}: pages, k and v must be {dt} like q; got {k_pages.dtype}, {v_pages.dtype}"
                        + ("" if k is None else f", {k.dtype}, {v.dtype}"))
    if not (k_pages.is_contiguous() and v_pages.is_contiguous()):
        raise ValueError(f"{who}: pages must be contiguous")
    if k is not None:
        want = (total, kvh, d) if packed else (n, rows, kvh, d)
        if k.shape != want or v.shape != want:
            raise ValueError(f"{who}: k / v must be {want}; got {tuple(k.shape)}, {tuple(v.shape)}")
    _native.inference_only(who, q, k_pages, v_pages, k, v, out)
    table = _i32(who, "table", table, (n, width))
    kv_lens = _i32(who, "kv_lens", kv_lens, (n,))
    if starts is not None:
        starts = _i32(who, "starts", starts, (n,))
    if out is not None and (out.shape != shape or out.dtype != dt or not out.is_contiguous()):
        raise ValueError(f"{who}: out must be a contiguous {tuple(shape)} {dt} tensor")
    dev = _native.device_index(who, (("q", q), ("k_pages", k_pages), ("v_pages", v_pages), ("k", k), ("v", v),
                                     ("table", table), ("kv_lens", kv_lens), ("starts", starts), ("offsets", offsets),
                                     ("out", out)))
    q, qs = _rows16(q)
    zero_tail = packed and out is None
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else torch.empty(shape, dtype=dt, device=q.device)
    if k is None:
        kp = vp = 0
        ks = vs = _NO_STRIDES
    else:
        (k, ks), (v, vs) = _rows16(k), _rows16(v)
        kp, vp = k.data_ptr(), v.data_ptr()
    if packed:
        qs, ks, vs = (0,) + qs, (0,) + ks[-3:], (0,) + vs[-3:]
    capacity = width * ps
    ptrs = (q.data_ptr(), kp, vp, k_pages.data_ptr(), v_pages.data_ptr(), out.data_ptr())
    fixed = (table.data_ptr(), kv_lens.data_ptr(), 0 if starts is None else starts.data_ptr(),
             offsets.data_ptr() if packed else 0, n, rows, total, heads, kvh, d, pages, ps, width,
             capacity if max_kv is None else min(int(max_kv), capacity), qs[0], qs[1], qs[2], ks[0], ks[1], ks[2],
             vs[0], vs[1], vs[2], tag, 1 if causal else 0, 1 if zero_tail else 0, d ** -0.5 if scale is None else scale)
    lib = _native.load_library()
    args = _ARGS.pack(*ptrs, 0, *fixed)
    need = lib.mfl_paged_attention_workspace_bytes(args)
    if need < 0:
        _error(who)
    with _native.on_device(dev):
        if need:
            ws = torch.empty(need, dtype=torch.uint8, device=q.device)
            args = _ARGS.pack(*ptrs, ws.data_ptr(), *fixed)
        if lib.mfl_paged_attention(args, _native.raw_stream(dev)) != 0:
            _error(who)
    return out


def _data(who, data):
    if data is None:
        return 0, 0, 0, 0
    if data.dim() != 6 or data.shape[1] != 2:
        raise ValueError(f"{who}: data must be (layers, 2, pages, kv_heads, page_size, dim); got {tuple(data.shape)}")
    _native.inference_only(who, data)
    if not data.is_contiguous():
        raise ValueError(f"{who}: data must be contiguous")
    row = data.shape[5] * data.element_size()
    if row % 16:
        raise ValueError(f"{who}: rows of {row} bytes (a multiple of 16)")
    return data.data_ptr(), data.shape[0] * 2, data.shape[3], row


def pages_update(data, table, lens, refs, *, parents=None, new_lens=None, page_size=None):
    """The next state of a page pool: every row a share of its parent's pages, cut or grown.

    data: (layers, 2, pages, kv_heads, page_size, dim) or None (``page_size`` then says how long a page is; a power of
    two up to 1024);
    table (n, width), lens (n), refs (pages), all int32.  Row s of the result holds what row ``parents[s]`` held
    (default: itself; outside [0, n): nothing) up to ``new_lens[s]`` tokens (default: all), and pages for the
    tokens up to new_lens[s] where that is more.  Full pages are shared; a row that grows inside a page that
    others keep gets its own copy of the used tokens in every layer.  Pages that nobody holds any more are free.
    New pages are the lowest free ones in row order.  Freeing a row: new_lens 0 (or parent -1).

    Returns (table, lens, refs, short), new tensors.  ``short`` (1) int32: 0, or how many pages are lacking —
    then nothing has changed.  ``data`` is changed in place (free pages only).
    """
    who = "pages_update"
    if table.dim() != 2:
        raise ValueError(f"{who}: table must be (n, width); got {tuple(table.shape)}")
    n, width = table.shape
    if refs.dim() != 1:
        raise ValueError(f"{who}: refs must be (pages,); got {tuple(refs.shape)}")
    pages = refs.shape[0]
    ptr, planes, heads, row = _data(who, data)
    if data is None:
        if page_size is None:
            raise ValueError(f"{who}: page_size is needed without data")
    else:
        if data.shape[2] != pages:
            raise ValueError(f"{who}: data has {data.shape[2]} pages, refs {pages}")
        if page_size is not None and page_size != data.shape[4]:
            raise ValueError(f"{who}: page_size {page_size}, data's pages hold {data.shape[4]}")
        page_size = data.shape[4]
    table = _i32(who, "table", table, (n, width))
    lens = _i32(who, "lens", lens, (n,))
    refs = _i32(who, "refs", refs, (pages,))
    if parents is not None:
        parents = _i32(who, "parents", parents, (n,))
    if new_lens is not None:
        new_lens = _i32(who, "new_lens", new_lens, (n,))
    dev = _native.device_index(who, (("table", table), ("lens", lens), ("refs", refs), ("parents", parents),
                                     ("new_lens", new_lens), ("data", data)))
    lib = _native.load_library()
    need = lib.mfl_pages_update_workspace_bytes(n, pages)
    with _native.on_device(dev):
        table_out, lens_out, refs_out = torch.empty_like(table), torch.empty_like(lens), torch.empty_like(refs)
        short = torch.empty(1, dtype=torch.int32, device=table.device)
        ws = torch.empty(need, dtype=torch.uint8, device=table.device)
        if lib.mfl_pages_update(table.data_ptr(), lens.data_ptr(), refs.data_ptr(),
                                None if parents is None else parents.data_ptr(),
                                None if new_lens is None else new_lens.data_ptr(), n, width, pages, page_size, ptr or None,
                                planes, heads, row, table_out.data_ptr(), lens_out.data_ptr(), refs_out.data_ptr(),
                                short.data_ptr(), ws.data_ptr(), _native.raw_stream(dev)) != 0:
            _error(who)
    return table_out, lens_out, refs_out, short


def pages_compact(data, table, refs):
    """Brings the live pages (refs > 0) to the front of the pool: with L of them, the k-th lowest live page at or
    behind L moves to the k-th lowest free page before L, in every layer.

    data as in ``pages_update`` (or None); table any int32 shape.  Returns (table, refs, remap, live), new tensors:
    remap (pages) int32 the new number of each page (-1: free), live (1) int32.  Table entries of free pages or
    outside the pool become -1.
    """
    who = "pages_compact"
    if refs.dim() != 1:
        raise ValueError(f"{who}: refs must be (pages,); got {tuple(refs.shape)}")
    pages = refs.shape[0]
    ptr, planes, heads, row = _data(who, data)
    page_bytes = 0
    if data is not None:
        if data.shape[2] != pages:
            raise ValueError(f"{who}: data has {data.shape[2]} pages, refs {pages}")
        page_bytes = heads * data.shape[4] * row
    table = _i32(who, "table", table, tuple(table.shape))
    refs = _i32(who, "refs", refs, (pages,))
    dev = _native.device_index(who, (("table", table), ("refs", refs), ("data", data)))
    lib = _native.load_library()
    with _native.on_device(dev):
        table_out, refs_out, remap = torch.empty_like(table), torch.empty_like(refs), torch.empty_like(refs)
        live = torch.empty(1, dtype=torch.int32, device=table.device)
        ws = torch.empty(lib.mfl_pages_compact_workspace_bytes(pages), dtype=torch.uint8, device=table.device)
        if lib.mfl_pages_compact(table.data_ptr(), table.numel(), refs.data_ptr(), pages, ptr or None, planes,
                                 page_bytes, table_out.data_ptr(), refs_out.data_ptr(), remap.data_ptr(),
                                 live.data_ptr(), ws.data_ptr(), _native.raw_stream(dev)) != 0:
            _error(who)
    return table_out, refs_out, remap, live


def pages_copy(data, src, dst):
    """Copies page src[i] to page dst[i] in every layer of ``data`` (in place).  src, dst: (count) int32; pairs with
    a number outside the pool are skipped.  No page may be both a source and a destination, or a destination
    twice (the result is then one of the possible ones)."""
    who = "pages_copy"
    if data is None:
        raise ValueError(f"{who}: data is needed")
    ptr, planes, heads, row = _data(who, data)
    if src.dim() != 1:
        raise ValueError(f"{who}: src must be (count,); got {tuple(src.shape)}")
    src = _i32(who, "src", src, (src.shape[0],))
    dst = _i32(who, "dst", dst, (src.shape[0],))
    dev = _native.device_index(who, (("data", data), ("src", src), ("dst", dst)))
    lib = _native.load_library()
    with _native.on_device(dev):
        if lib.mfl_pages_copy(src.data_ptr(), dst.data_ptr(), src.shape[0], ptr, planes, data.shape[2],
                              heads * data.shape[4] * row, _native.raw_stream(dev)) != 0:
            _error(who)
    return data


class PagedKVCache:
    """The paged keys and values of ``rows`` sequences of up to ``max_tokens`` tokens, all layers.

    data (layers, 2, pages, kv_heads, page_size, head_dim); table (rows, width), lens (rows), refs (pages) int32 —
    the state that the functions above take and return; ``short`` (1) int32 is the last update's.  With the
    default number of pages no update can run short."""

    def __init__(self, layers, rows, max_tokens, kv_heads, head_dim, page_size=16, pages=None, dtype=torch.bfloat16,
                 device="cuda"):
        if page_size < 1 or page_size > 1024 or page_size & (page_size - 1):
            raise ValueError(f"PagedKVCache: page_size {page_size} is no power of two up to 1024")
        self.page_size, self.max_tokens = page_size, max_tokens
        width = max(1, (max_tokens + page_size - 1) // page_size)
        pages = rows * width if pages is None else pages  # (no rows can hold more different ones)
        self.data = torch.zeros(layers, 2, pages, kv_heads, page_size, head_dim, dtype=dtype, device=device)
        self.table = torch.full((rows, width), -1, dtype=torch.int32, device=device)
        self.lens = torch.zeros(rows, dtype=torch.int32, device=device)
        self.refs = torch.zeros(pages, dtype=torch.int32, device=device)
        self.short = torch.zeros(1, dtype=torch.int32, device=device)

    def update(self, parents=None, new_lens=None):
        """``pages_update`` of the whole cache.  The state becomes new tensors: a captured update reads those of its
        capture at every replay, so steps that follow each other copy the results back into them (or are one graph)."""
        self.table, self.lens, self.refs, self.short = pages_update(
            self.data, self.table, self.lens, self.refs, parents=parents, new_lens=new_lens)

    def compact(self):
        """``pages_compact`` of the whole cache; returns the number of live pages, (1) int32."""
        self.table, self.refs, _, live = pages_compact(self.data, self.table, self.refs)
        return live

    def attend(self, layer, q, k=None, v=None, **kw):
        """``paged_attention`` over one layer."""
        kw.setdefault("max_kv", self.max_tokens)
        return paged_attention(q, self.data[layer, 0], self.data[layer, 1], self.table, self.lens, k=k, v=v, **kw)

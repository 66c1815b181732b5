"""Pages of a KV cache: reserve, free, fork, copy, and moving kept rows together (additions of this library; the reference's
cache calls take a page table as it is given, flash_attn_npu_3/flash_attn_npu_interface.py:965).

The pool's state is one int32 reference count a page, `page_refs` (num_pages,), zeros to begin with; a page is free when its
count is 0.  Page tables are int32 (batch, max_pages), filled from the left, -1 where there is no page.  Everything stays on
the device and on the current stream: no call waits for the host, and each can be captured into a CUDA graph."""
import functools
import struct
from typing import Optional

import torch

import fa_b200_capi as capi

_VIEW = struct.Struct("=Qqqqqiii4x")
assert _VIEW.size == capi.C.sizeof(capi.CacheView)


def _int32(name, t, dims, index):
    """Checks of an int32 tensor -> its shape.  A small call's kernels run 2 to 10 us: tensors are asked as little as possible."""
    if not isinstance(t, torch.Tensor) or t.dtype is not torch.int32:
        raise RuntimeError(f"{name} must be an int32 tensor")
    if t.get_device() != index:
        capi.cuda_index(t)
        raise RuntimeError(f"{name} must be on the device of the other tensors")
    shape = t.shape
    if len(shape) != dims:
        raise RuntimeError(f"{name} must have shape with {dims} dimension{'s' if dims > 1 else ''}, not {tuple(shape)}")
    return shape


def _row(name, t, n, index):
    """An input (n,) -> a dense tensor."""
    if _int32(name, t, 1, index)[0] != n:
        raise RuntimeError(f"{name} must have shape {(n,)}, not {tuple(t.shape)}")
    return t if t.is_contiguous() else t.contiguous()


def _read_table(name, t, b, index):
    """An input (b, any), b None: any -> (tensor, its shape, distance of its rows); a copy where its last dimension is strided."""
    shape = _int32(name, t, 2, index)
    if b is not None and shape[0] != b:
        raise RuntimeError(f"{name} must have shape {(b, 'any')}, not {tuple(shape)}")
    st = t.stride()
    if st[1] != 1:
        t = t.contiguous()
        st = t.stride()
    return t, shape, st[0]


def _written_table(name, t, index):
    """A table that is changed in place -> (b, width, distance of its rows)."""
    b, width = _int32(name, t, 2, index)
    s0, s1 = t.stride()
    if (s1 != 1 and width > 1) or (b > 1 and s0 < width):
        raise RuntimeError(f"{name} is changed in place: its last dimension must be contiguous and its rows apart")
    return b, width, s0


def _pool(page_refs):
    """-> (device number, pages)"""
    if not isinstance(page_refs, torch.Tensor):
        raise RuntimeError("page_refs must be an int32 tensor")
    index = capi.cuda_index(page_refs)
    pages = _int32("page_refs", page_refs, 1, index)[0]
    if not page_refs.is_contiguous():
        raise RuntimeError("page_refs is changed in place: it must be contiguous")
    if not 0 < pages <= 1 << 24:
        raise RuntimeError("page_refs must have 1 to 2^24 entries")
    return index, pages


def _views(caches):
    """Caches -> (packed fa_cache_view array, how many, entries, rows of one, device number).  A tensor of up to four dimensions
    is one cache (entries, rows, [heads,] [dim]); one of five is a stack of caches."""
    caches = (caches,) if isinstance(caches, torch.Tensor) else tuple(caches)
    if not caches:
        raise RuntimeError("at least one cache is needed")
    pack, size_of = _VIEW.pack_into, _VIEW.size
    buf = (capi.C.c_char * (size_of * len(caches)))()
    entries = rows = index = None
    at = 0
    for c in caches:
        if not isinstance(c, torch.Tensor):
            raise RuntimeError("caches must be tensors")
        shape, st, size = c.shape, c.stride(), c.element_size()
        dims = len(shape)
        n, sc = 1, 0
        if dims == 5:
            n, sc = shape[0], st[0]
            shape, st = shape[1:], st[1:]
        elif not 2 <= dims <= 4:
            raise RuntimeError("a cache must be a tensor (num_pages, page_size, [nheads,] [headdim]), or a stack of such with five dimensions")
        heads, sh, dim = (shape[2], st[2], shape[3]) if dims >= 4 else (1, 0, shape[2] if dims == 3 else 1)
        if dims > 2 and st[-1] != 1:
            raise RuntimeError("caches must have a contiguous last dimension")
        if index is None:
            entries, rows, index = shape[0], shape[1], capi.cuda_index(c)
        elif shape[0] != entries or shape[1] != rows or c.get_device() != index:
            capi.cuda_index(c)
            raise RuntimeError("all caches must have the same number of pages, the same page size and the same device")
        if n * entries * rows * heads * dim == 0:
            raise RuntimeError("a cache is empty")
        if (n > 1 and sc == 0) or (st[0] == 0 and entries > 1) or (st[1] == 0 and rows > 1) or (heads > 1 and sh == 0):
            raise RuntimeError("caches may not be expanded")
        pack(buf, at, c.data_ptr(), sc * size, st[0] * size, st[1] * size, sh * size, n, heads, dim * size)
        at += size_of
    return buf, len(caches), entries, rows, index


def _sizes(extra, page_size):
    if type(extra) is not int or not 0 <= extra < 2 ** 31:
        raise RuntimeError("extra must be a non-negative integer")
    if type(page_size) is not int or not 0 < page_size < 2 ** 31:
        raise RuntimeError("page_size must be a positive integer")


def _run(fn, index, views, num_caches, num_pages, page_size, refs, table, table_stride, b, width, extra, n, keep_parents, seqlens, rows,
         rows2, rows_stride, batch_idx, new_table, new_seqlens, missing, ws=None):
    """The library call: tensors, or None, where the block takes pointers."""
    p = [0 if t is None else t.data_ptr() for t in (refs, table, seqlens, rows, rows2, batch_idx, new_table, new_seqlens, missing, ws)]
    buf = capi.PAGES_BLOCK.new(
        0 if views is None else capi.C.addressof(views), num_caches, num_pages, page_size, p[0], p[1], table_stride, b, width, extra, n,
        keep_parents, p[2], p[3], p[4], rows_stride, p[5], p[6], p[7], p[8], p[9], 0 if ws is None else ws.numel() * 4, capi.raw_stream_of(index))
    capi.launch_on(fn, buf, index)


@functools.lru_cache(maxsize=256)
def _workspace_ints(rows, num_pages):
    return (capi.lib.fa_pages_workspace_bytes(rows, num_pages) + 3) // 4


def _workspace(like, rows, num_pages):
    return like.new_empty(_workspace_ints(rows, num_pages))


def kvcache_reserve(page_refs, page_table, cache_seqlens, page_size, extra=0):
    """Give every sequence the pages that cache_seqlens + extra rows need, in place: entries of page_table below that which are
    -1 get the lowest free pages, rows in order and entries in order, with a count of 1.  cache_seqlens int32 (batch,).
    Rows that need more pages than the table is wide get what fits.  Returns `missing`, int32 (1,): entries that stayed -1
    because no page was free."""
    index, pages = _pool(page_refs)
    _sizes(extra, page_size)
    b, width, stride = _written_table("page_table", page_table, index)
    lens = _row("cache_seqlens", cache_seqlens, b, index)
    missing = page_refs.new_empty(1)
    _run(capi._call_reserve, index, None, 0, pages, page_size, page_refs, page_table, stride, b, width, extra, 0, 0, lens, None, None, 0, None,
         None, None, missing, _workspace(page_refs, b, pages))
    return missing


def kvcache_free(page_refs, page_table, cache_seqlens: Optional[torch.Tensor] = None, page_size=None, extra=0):
    """Let go of the pages behind cache_seqlens + extra rows (of all pages when cache_seqlens is None; page_size is only needed
    with it), in place: their counts drop by one and their entries of page_table become -1.  A page whose count is 0 stays at 0."""
    index, pages = _pool(page_refs)
    b, width, stride = _written_table("page_table", page_table, index)
    if cache_seqlens is None:
        page_size, extra, lens = 1, 0, None
    else:
        _sizes(extra, page_size)
        lens = _row("cache_seqlens", cache_seqlens, b, index)
    _run(capi._call_free, index, None, 0, pages, page_size, page_refs, page_table, stride, b, width, extra, 0, 0, lens, None, None, 0, None,
         None, None, None)


def kvcache_fork(caches, page_refs, page_table, cache_seqlens, parents, keep_parents=False):
    """Continue sequences several times: beam search, parallel samples.

    Row i of the new table continues row parents[i] (int32 (n,), n at most 2^20) of page_table; a number outside it makes an empty row.  Full
    pages are shared, their counts grow.  Of the rows that hold the same partly filled last page, the last keeps it, and the
    others get a copy of its rows in the lowest free pages, in all caches; all of them do when somebody else holds it too.
    With keep_parents the old rows stay valid (and hold their pages); without, they let go of theirs, as when beams are
    reordered: use the new table instead.  Entries behind the length are -1.

    caches: a tensor or a list of tensors (num_pages, page_size, nheads, headdim) (also without the last or the last two
    dimensions, such as scales), or of five dimensions, a stack of such.  cache_seqlens int32 (batch,).
    Returns (page_table (n, max_pages), cache_seqlens (n,), missing (1,)): rows whose copy found no free page end with their
    last full page and are counted in `missing`."""
    index, pages = _pool(page_refs)
    views, num, entries, page_size, device = _views(caches)
    if entries != pages or device != index:
        raise RuntimeError("page_refs must have one entry for every page of the caches, on their device")
    table, (b, width), stride = _read_table("page_table", page_table, None, index)
    lens = _row("cache_seqlens", cache_seqlens, b, index)
    n = _int32("parents", parents, 1, index)[0]
    if not parents.is_contiguous():
        parents = parents.contiguous()
    new_table = page_refs.new_empty((n, width))
    new_lens, missing = torch.empty_like(parents), page_refs.new_empty(1)
    _run(capi._call_fork, index, views, num, pages, page_size, page_refs, table, stride, b, width, 0, n, 1 if keep_parents else 0, lens, parents,
         None, 0, None, new_table, new_lens, missing, _workspace(page_refs, n, pages))
    return new_table, new_lens, missing


def kvcache_copy_pages(caches, src, dst):
    """Copy page src[i] to page dst[i] (int32 (n,)) in all caches (as in kvcache_fork).  Pairs with a page outside the cache
    are skipped.  A page that is written may not stand anywhere else in the lists."""
    views, num, pages, page_size, index = _views(caches)
    n = _int32("src", src, 1, index)[0]
    src, dst = _row("src", src, n, index), _row("dst", dst, n, index)
    _run(capi._call_copy, index, views, num, pages, page_size, None, None, 0, 0, 0, 0, n, 0, None, src, dst, 0, None, None, None, None)


def kvcache_compact(caches, cache_seqlens, kept, counts: Optional[torch.Tensor] = None, page_table: Optional[torch.Tensor] = None,
                    cache_batch_idx: Optional[torch.Tensor] = None):
    """Keep some of the rows behind cache_seqlens and move them together: the accepted tokens of a draft.

    Row cache_seqlens[b] + kept[b, i] of sequence b becomes row cache_seqlens[b] + i, for i < counts[b], in all caches (as in
    kvcache_fork; without page_table dense caches (batch_cache, seqlen_cache, nheads, headdim), whose entry of a sequence
    cache_batch_idx may name).  kept int32 (batch, n), strictly increasing in each row; counts int32 (batch,), None: n.  A
    sequence's list ends at the first entry that is not larger than the one before, or negative, or past the capacity.  The
    rows that move must lie on pages (or in cache entries) that no other sequence holds, and the caches may share no memory; a
    row on a page that is not in the cache is left out of the move.  cache_seqlens of zeros prunes whole sequences.  Returns the new lengths, int32 (batch,)."""
    views, num, entries, rows, index = _views(caches)
    b = _int32("cache_seqlens", cache_seqlens, 1, index)[0]
    lens = cache_seqlens if cache_seqlens.is_contiguous() else cache_seqlens.contiguous()
    kept, (_, n), kept_stride = _read_table("kept", kept, b, index)
    if counts is not None:
        counts = _row("counts", counts, b, index)
    table, width, stride = None, 1, 0
    if page_table is not None:
        if cache_batch_idx is not None:
            raise RuntimeError("cache_batch_idx is not used with a paged cache")
        table, (_, width), stride = _read_table("page_table", page_table, b, index)
        if width == 0:
            raise RuntimeError("page_table has no entries")
    elif cache_batch_idx is not None:
        cache_batch_idx = _row("cache_batch_idx", cache_batch_idx, b, index)
    elif entries < b:
        raise RuntimeError("the caches have fewer entries than the batch")
    out = torch.empty_like(lens)
    _run(capi._call_compact, index, views, num, entries, rows, None, table, stride, b, width, 0, n, 0, lens, kept, counts, kept_stride,
         cache_batch_idx, None, out, None)
    return out

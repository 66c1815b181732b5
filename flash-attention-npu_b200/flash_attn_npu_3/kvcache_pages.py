"""Pages of a KV cache: reserve, free, fork, copy, and moving kept rows together (additions of this library; the reference's
cache calls take a page table as it is given, flash_attn_npu_3/flash_attn_npu_interface.py:965).

The pool's state is one int32 reference count a page, `page_refs` (num_pages,), zeros to begin with; a page is free when its
count is 0.  Page tables are int32 (batch, max_pages), filled from the left, -1 where there is no page.  Everything stays on
the device and on the current stream: no call waits for the host, and each can be captured into a CUDA graph."""
import struct
from typing import Optional

import torch

import fa_b200_capi as capi

_VIEW = struct.Struct("=Qqqqqiii4x")
assert _VIEW.size == capi.C.sizeof(capi.CacheView)


def _int32(name, t, shape, device=None):
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32:
        raise RuntimeError(f"{name} must be an int32 tensor")
    if not t.is_cuda:
        raise RuntimeError("expected CUDA tensors: this library has no CPU implementation")
    if device is not None and t.device != device:
        raise RuntimeError(f"{name} must be on the device of the other tensors")
    if len(shape) != t.dim() or any(s is not None and s != n for s, n in zip(shape, t.shape)):
        raise RuntimeError(f"{name} must have shape {tuple('any' if s is None else s for s in shape)}, not {tuple(t.shape)}")
    return t


def _read(name, t, shape, device=None):
    """An input: a copy where its last dimension is strided."""
    t = _int32(name, t, shape, device)
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def _written(name, t, shape, device=None):
    """A tensor that is changed in place."""
    t = _int32(name, t, shape, device)
    s = t.stride()
    if (s[-1] != 1 and t.shape[-1] > 1) or (len(s) == 2 and t.shape[0] > 1 and s[0] < t.shape[1]):
        raise RuntimeError(f"{name} is changed in place: its last dimension must be contiguous and its rows apart")
    return t


def _views(caches):
    """Caches -> (packed fa_cache_view array, how many, entries, rows of one, device).  A tensor of up to four dimensions is one
    cache (entries, rows, [heads,] [dim]); one of five is a stack of caches."""
    caches = [caches] if isinstance(caches, torch.Tensor) else list(caches)
    if not caches:
        raise RuntimeError("at least one cache is needed")
    entries = rows = device = None
    buf = bytearray(_VIEW.size * len(caches))
    for i, c in enumerate(caches):
        if not isinstance(c, torch.Tensor) or not 2 <= c.dim() <= 5:
            raise RuntimeError("a cache must be a tensor (num_pages, page_size, [nheads,] [headdim]), or a stack of such with five dimensions")
        if not c.is_cuda:
            raise RuntimeError("expected CUDA tensors: this library has no CPU implementation")
        size, shape, st = c.element_size(), tuple(c.shape), c.stride()
        n, sc = 1, 0
        if len(shape) == 5:
            n, sc = shape[0], st[0]
            shape, st = shape[1:], st[1:]
        heads, sh, dim = (shape[2], st[2], shape[3]) if len(shape) == 4 else (1, 0, shape[2] if len(shape) == 3 else 1)
        if len(shape) > 2 and st[-1] != 1:
            raise RuntimeError("caches must have a contiguous last dimension")
        if (n > 1 and sc == 0) or st[0] == 0 and shape[0] > 1 or st[1] == 0 and shape[1] > 1 or heads > 1 and sh == 0:
            raise RuntimeError("caches may not be expanded")
        if i == 0:
            entries, rows, device = shape[0], shape[1], c.device
        elif (shape[0], shape[1]) != (entries, rows) or c.device != device:
            raise RuntimeError("all caches must have the same number of pages, the same page size and the same device")
        if c.numel() == 0:
            raise RuntimeError("a cache is empty")
        _VIEW.pack_into(buf, i * _VIEW.size, c.data_ptr(), sc * size, st[0] * size, st[1] * size, sh * size, n, heads, dim * size)
    return buf, len(caches), entries, rows, device


def _launch(fn, device, views=None, num_views=0, num_pages=0, page_size=0, refs=None, table=None, b=0, width=0, extra=0, n=0,
            keep_parents=0, seqlens=None, rows=None, rows2=None, rows_stride=0, batch_idx=None, new_table=None, new_seqlens=None,
            missing=None, workspace_rows=None):
    p = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    ws, nbytes = None, 0
    if workspace_rows is not None:
        nbytes = capi.lib.fa_pages_workspace_bytes(workspace_rows, num_pages)
        ws = capi.workspace(nbytes, device)
    host = (capi.C.c_char * len(views)).from_buffer(views) if views is not None else None
    buf = capi.PAGES_BLOCK.new(
        0 if host is None else capi.C.addressof(host), num_views, num_pages, page_size, p(refs), p(table), 0 if table is None else table.stride(0),
        b, width, extra, n, keep_parents, p(seqlens), p(rows), p(rows2), rows_stride, p(batch_idx), p(new_table), p(new_seqlens), p(missing),
        p(ws), nbytes, capi.raw_stream(device))
    capi.launch(fn, buf, device)


def _extra(extra, page_size):
    if type(extra) is not int or not 0 <= extra < 2 ** 31:
        raise RuntimeError("extra must be a non-negative integer")
    if type(page_size) is not int or not 0 < page_size < 2 ** 31:
        raise RuntimeError("page_size must be a positive integer")


def _pool(page_refs):
    refs = _written("page_refs", page_refs, (None,))
    if not 0 < refs.shape[0] <= 1 << 24:
        raise RuntimeError("page_refs must have 1 to 2^24 entries")
    return refs


def kvcache_reserve(page_refs, page_table, cache_seqlens, page_size, extra=0):
    """Give every sequence the pages that cache_seqlens + extra rows need, in place: entries of page_table below that which are
    -1 get the lowest free pages, rows in order and entries in order, with a count of 1.  cache_seqlens int32 (batch,).
    Rows that need more pages than the table is wide get what fits.  Returns `missing`, int32 (1,): entries that stayed -1
    because no page was free."""
    refs = _pool(page_refs)
    _extra(extra, page_size)
    table = _written("page_table", page_table, (None, None), refs.device)
    b, width = table.shape
    lens = _read("cache_seqlens", cache_seqlens, (b,), refs.device)
    missing = torch.empty((1,), dtype=torch.int32, device=refs.device)
    _launch(capi._call_reserve, refs.device, num_pages=refs.shape[0], page_size=page_size, refs=refs, table=table, b=b, width=width,
            extra=extra, seqlens=lens, missing=missing, workspace_rows=b)
    return missing


def kvcache_free(page_refs, page_table, cache_seqlens: Optional[torch.Tensor] = None, page_size=None, extra=0):
    """Let go of the pages behind cache_seqlens + extra rows (of all pages when cache_seqlens is None; page_size is only needed
    with it), in place: their counts
    drop by one and their entries of page_table become -1.  A page whose count is 0 stays at 0."""
    refs = _pool(page_refs)
    if cache_seqlens is None:
        page_size, extra = 1, 0
    _extra(extra, page_size)
    table = _written("page_table", page_table, (None, None), refs.device)
    b, width = table.shape
    lens = None if cache_seqlens is None else _read("cache_seqlens", cache_seqlens, (b,), refs.device)
    _launch(capi._call_free, refs.device, num_pages=refs.shape[0], page_size=page_size, refs=refs, table=table, b=b, width=width,
            extra=extra, seqlens=lens)


def kvcache_fork(caches, page_refs, page_table, cache_seqlens, parents, keep_parents=False):
    """Continue sequences several times: beam search, parallel samples.

    Row i of the new table continues row parents[i] (int32 (n,)) of page_table; a number outside it makes an empty row.  Full
    pages are shared, their counts grow.  Of the rows that hold the same partly filled last page, the last keeps it, and the
    others get a copy of its rows in the lowest free pages, in all caches; all of them do when somebody else holds it too.
    With keep_parents the old rows stay valid (and hold their pages); without, they let go of theirs, as when beams are
    reordered: use the new table instead.  Entries behind the length are -1.

    caches: a tensor or a list of tensors (num_pages, page_size, nheads, headdim) (also without the last or the last two
    dimensions, such as scales), or of five dimensions, a stack of such.  cache_seqlens int32 (batch,).
    Returns (page_table (n, max_pages), cache_seqlens (n,), missing (1,)): rows whose copy found no free page end with their
    last full page and are counted in `missing`."""
    refs = _pool(page_refs)
    views, num, pages, page_size, device = _views(caches)
    if pages != refs.shape[0] or refs.device != device:
        raise RuntimeError("page_refs must have one entry for every page of the caches, on their device")
    table = _read("page_table", page_table, (None, None), device)
    b, width = table.shape
    lens = _read("cache_seqlens", cache_seqlens, (b,), device)
    parents = _read("parents", parents, (None,), device)
    n = parents.shape[0]
    new_table = torch.empty((n, width), dtype=torch.int32, device=device)
    new_lens = torch.empty((n,), dtype=torch.int32, device=device)
    missing = torch.empty((1,), dtype=torch.int32, device=device)
    _launch(capi._call_fork, device, views, num, pages, page_size, refs, table, b, width, 0, n, int(bool(keep_parents)), lens, parents,
            new_table=new_table, new_seqlens=new_lens, missing=missing, workspace_rows=n)
    return new_table, new_lens, missing


def kvcache_copy_pages(caches, src, dst):
    """Copy page src[i] to page dst[i] (int32 (n,)) in all caches (as in kvcache_fork).  Pairs with a page outside the cache
    are skipped.  A page that is written may not stand anywhere else in the lists."""
    views, num, pages, page_size, device = _views(caches)
    src = _read("src", src, (None,), device)
    dst = _read("dst", dst, (src.shape[0],), device)
    _launch(capi._call_copy, device, views, num, pages, page_size, n=src.shape[0], rows=src, rows2=dst)


def kvcache_compact(caches, cache_seqlens, kept, counts: Optional[torch.Tensor] = None, page_table: Optional[torch.Tensor] = None,
                    cache_batch_idx: Optional[torch.Tensor] = None):
    """Keep some of the rows behind cache_seqlens and move them together: the accepted tokens of a draft.

    Row cache_seqlens[b] + kept[b, i] of sequence b becomes row cache_seqlens[b] + i, for i < counts[b], in all caches (as in
    kvcache_fork; without page_table dense caches (batch_cache, seqlen_cache, nheads, headdim), whose entry of a sequence
    cache_batch_idx may name).  kept int32 (batch, n), strictly increasing in each row; counts int32 (batch,), None: n.  A
    sequence's list ends at the first entry that is not larger than the one before, or negative, or past the capacity.  The
    rows that move must lie on pages that no other sequence holds; a row on a page that is not in the cache is left out of
    the move.  cache_seqlens of zeros prunes whole sequences.  Returns the new lengths, int32 (batch,)."""
    views, num, pages, page_size, device = _views(caches)
    lens = _read("cache_seqlens", cache_seqlens, (None,), device)
    b = lens.shape[0]
    kept = _read("kept", kept, (b, None), device)
    counts = None if counts is None else _read("counts", counts, (b,), device)
    table, width = None, 1
    if page_table is not None:
        if cache_batch_idx is not None:
            raise RuntimeError("cache_batch_idx is not used with a paged cache")
        table = _read("page_table", page_table, (b, None), device)
        width = table.shape[1]
        if width == 0:
            raise RuntimeError("page_table has no entries")
    elif cache_batch_idx is not None:
        cache_batch_idx = _read("cache_batch_idx", cache_batch_idx, (b,), device)
    elif pages < b:
        raise RuntimeError("the caches have fewer entries than the batch")
    out = torch.empty((b,), dtype=torch.int32, device=device)
    _launch(capi._call_compact, device, views, num, pages, page_size, table=table, b=b, width=width, n=kept.shape[1], seqlens=lens,
            rows=kept, rows2=counts, rows_stride=kept.stride(0), batch_idx=cache_batch_idx, new_seqlens=out)
    return out

"""Pages of a paged KV cache: copied, forked with copy on write, compacted and
listed as free (the reference's drivers build one fixed page table).

The page table ``(kv_page_indptr, kv_page_indices, kv_last_page_len)`` of the
paged decodes is the only record: a page is live when the table names it, or
when the optional ``reserved`` mask (``[num_pages]`` bool: pages that another
holder keeps, a prefix store's say, named by the table or not) marks it.  Every call below takes the table
of the whole pool and returns a new one; the old table stays valid for what was
launched before.  Dropping a sequence is leaving it out; there are no reference
counts.  The pool is ``[num_pages, 2, Hkv, page_size, D]``, or
``[num_layers, num_pages, 2, Hkv, page_size, D]`` with one table for all layers.
Runs on torch's current stream (sm_100a, ``csrc/pages.cu``).
"""
from __future__ import annotations

import torch

from . import _lib


_TYPES = (torch.float16, torch.bfloat16)
_copy = _lib.Entry("akt_copy_kv_pages", _lib.PagePool, _lib.c_void_p, _lib.c_void_p, _lib.c_int64, _lib.c_void_p)
_fork_size = _lib.Entry("akt_fork_paged_workspace_size", _lib.ForkPagedArgs, restype=_lib.c_size_t)
_fork = _lib.Entry("akt_fork_paged", _lib.ForkPagedArgs, _lib.c_void_p, _lib.c_size_t, _lib.c_void_p)
_compact_size = _lib.Entry("akt_compact_paged_workspace_size", _lib.CompactPagedArgs, restype=_lib.c_size_t)
_compact = _lib.Entry("akt_compact_paged", _lib.CompactPagedArgs, _lib.c_void_p, _lib.c_size_t, _lib.c_void_p)


def _pool(cache):
    """The fields of ``akt_page_pool``."""
    shape, stride = cache.shape, cache.stride()
    if len(shape) not in (5, 6) or shape[-4] != 2:
        raise ValueError("paged_kv_cache must be [num_pages, 2, Hkv, page_size, D], with layers before it or not")
    if cache.dtype not in _TYPES:
        raise TypeError(f"unsupported dtype {cache.dtype}: float16 or bfloat16 expected")
    layers, step = (shape[0], stride[0]) if len(shape) == 6 else (1, 0)
    return (cache.data_ptr(), step, *stride[-5:], shape[-5], layers, *shape[-3:])


def _reserved(mask, num_pages, like):
    if mask is None:
        return None
    if mask.dtype not in (torch.bool, torch.uint8) or mask.device != like.device or mask.shape != (num_pages,):
        raise ValueError("reserved must be a bool (or uint8) mask [num_pages] on the pool's device")
    return mask.contiguous()


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def copy_kv_pages(paged_kv_cache, src_pages, dst_pages):
    """Copy page ``src_pages[i]`` to page ``dst_pages[i]`` in every layer, in place.  No
    destination may be the source or destination of another copy."""
    index = _lib.device_index(paged_kv_cache)
    pool = _pool(paged_kv_cache)
    src, dst = _lib.list_i32(src_pages, paged_kv_cache), _lib.list_i32(dst_pages, paged_kv_cache)
    if src.dim() != 1 or src.shape != dst.shape:
        raise ValueError("src_pages and dst_pages must be lists of the same length")
    with _lib.on_index(index):
        _lib.check(_copy(pool, src.data_ptr(), dst.data_ptr(), src.numel(), _lib.raw_stream(index)))
    return paged_kv_cache


def fork_paged_kv_cache(paged_kv_cache, kv_page_indptr, kv_page_indices, kv_last_page_len, parents, reserved=None,
                        max_entries=None):
    """A new batch of sequences: child ``c`` continues sequence ``parents[c]``.

    Full pages are shared.  A partly filled last page, which the child will append to, goes
    over to the first child that ends in it, unless ``reserved`` marks it (a prefix that a
    store keeps) or a named parent has it as a full page (a sibling cut back into it); every
    other child gets its own copy, in the lowest-numbered pages that neither a named parent
    nor ``reserved`` holds.  Sequences that no child names are dropped.  So beam search's
    reordering, several samples of one prompt and dropping finished sequences (``parents`` =
    those that stay) are all this call.

    parents: [num_children] (int32)
    max_entries: length of the returned index array (``sum`` of the children's pages; a
        longer one is -1 past its end).  None: computed, which costs one device-to-host read
    returns (kv_page_indptr [num_children + 1], kv_page_indices [max_entries],
        kv_last_page_len [num_children]), int32
    """
    index = _lib.device_index(paged_kv_cache)
    pool = _pool(paged_kv_cache)
    indptr, indices = _lib.list_i32(kv_page_indptr, paged_kv_cache), _lib.list_i32(kv_page_indices, paged_kv_cache)
    last, par = _lib.list_i32(kv_last_page_len, paged_kv_cache), _lib.list_i32(parents, paged_kv_cache)
    B, F = indptr.numel() - 1, par.numel()
    if B < 0 or last.numel() != B or par.dim() != 1:
        raise ValueError("kv_page_indptr must have B+1 entries, kv_last_page_len B entries and parents be a list")
    mask = _reserved(reserved, pool[7], paged_kv_cache)
    if max_entries is None:
        at = par.long().clamp(0, max(B - 1, 0))
        max_entries = int((indptr[at + 1] - indptr[at]).sum()) if B and F else 0
    if max_entries < 0:
        raise ValueError("max_entries must not be negative")
    head = (*pool, indptr.data_ptr(), indices.data_ptr(), last.data_ptr(), indices.numel(), par.data_ptr(), _ptr(mask))
    size = _fork_size((*head, 0, 0, 0, max_entries, B, F))
    # the new table in one allocation; the workspace has its own, which goes when the call ends
    ws = indptr.new_empty(size // 4)
    out_indptr, out_indices, out_last = indptr.new_empty(2 * F + 1 + max_entries).split_with_sizes((F + 1, max_entries, F))
    with _lib.on_index(index):
        rc = _fork((*head, out_indptr.data_ptr(), out_indices.data_ptr(), out_last.data_ptr(), max_entries, B, F),
                   ws.data_ptr(), size, _lib.raw_stream(index))
        if rc:
            _lib.check(rc)
    return out_indptr, out_indices, out_last


def compact_paged_kv_cache(paged_kv_cache, kv_page_indices, reserved=None):
    """Move the live pages to the lowest page numbers that ``reserved`` leaves open, in
    place, so that the pool's tail is free.

    returns (kv_page_indices of the same length, pages_used): ``pages_used`` (int32 scalar
    on the device) is one past the highest page then in use or reserved.  ``kv_page_indptr``
    and ``kv_last_page_len`` stay as they are.
    """
    index = _lib.device_index(paged_kv_cache)
    pool = _pool(paged_kv_cache)
    indices = _lib.list_i32(kv_page_indices, paged_kv_cache)
    if indices.dim() != 1:
        raise ValueError("kv_page_indices must be a list")
    n = indices.shape[0]
    mask = _reserved(reserved, pool[7], paged_kv_cache)
    head = (*pool, indices.data_ptr(), n, _ptr(mask))
    size = _compact_size((*head, 0, 0))
    # the new index array and the count in one allocation; the workspace has its own, which goes when the call ends
    ws = indices.new_empty(size // 4)
    out, used = indices.new_empty(n + 1).split_with_sizes((n, 1))
    with _lib.on_index(index):
        rc = _compact((*head, out.data_ptr(), used.data_ptr()), ws.data_ptr(), size, _lib.raw_stream(index))
        if rc:
            _lib.check(rc)
    return out, used.view(())


def free_kv_pages(num_pages, kv_page_indices, reserved=None):
    """The pages that the table does not name, ascending: ``(pages [num_pages] int32, -1 past
    their count; count, int32 scalar on the device)``."""
    index = _lib.device_index(kv_page_indices)
    indices = _lib.list_i32(kv_page_indices, kv_page_indices)
    mask = _reserved(reserved, num_pages, indices)
    i32 = dict(dtype=torch.int32, device=indices.device)
    out, count = torch.empty(num_pages, **i32), torch.empty((), **i32)
    L = _lib.lib()
    with _lib.on_index(index):
        ws = _lib.workspace(L.akt_free_kv_pages_workspace_size(num_pages), indices.device)
        _lib.check(L.akt_free_kv_pages(indices.data_ptr(), indices.numel(), _ptr(mask), num_pages, out.data_ptr(),
                                       count.data_ptr(), ws.data_ptr(), ws.numel(), _lib.raw_stream(index)))
    return out, count

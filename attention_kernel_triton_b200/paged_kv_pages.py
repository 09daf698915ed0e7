"""Pages of a paged KV cache: copied, forked with copy on write, compacted and
listed as free (the reference's drivers build one fixed page table).

The page table ``(kv_page_indptr, kv_page_indices, kv_last_page_len)`` of the
paged decodes is the only record: a page is live when the table names it, or
when the optional ``reserved`` mask (``[num_pages]`` bool: pages that another
holder keeps, a prefix store's say) marks it.  Every call below takes the table
of the whole pool and returns a new one; the old table stays valid for what was
launched before.  Dropping a sequence is leaving it out; there are no reference
counts.  The pool is ``[num_pages, 2, Hkv, page_size, D]``, or
``[num_layers, num_pages, 2, Hkv, page_size, D]`` with one table for all layers.
Runs on torch's current stream (sm_100a, ``csrc/pages.cu``).
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib


def _pool(cache) -> _lib.PagePool:
    if cache.dim() not in (5, 6) or cache.shape[-4] != 2:
        raise ValueError("paged_kv_cache must be [num_pages, 2, Hkv, page_size, D], with layers before it or not")
    if cache.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"unsupported dtype {cache.dtype}: float16 or bfloat16 expected")
    q = _lib.PagePool()
    q.kv_cache = cache.data_ptr()
    stride = cache.stride()
    q.num_layers = cache.shape[0] if cache.dim() == 6 else 1
    q.stride_layer = stride[0] if cache.dim() == 6 else 0
    q.stride_page, q.stride_kv, q.stride_head, q.stride_token, q.stride_dim = stride[-5:]
    q.num_pages, q.num_kv_heads, q.page_size, q.head_dim = cache.shape[-5], *cache.shape[-3:]
    return q


def _i32(t, dev):
    return _lib.as_int32(t, dev).contiguous()


def _reserved(mask, num_pages, dev):
    if mask is None:
        return None
    if mask.dtype not in (torch.bool, torch.uint8) or mask.device != dev or mask.shape != (num_pages,):
        raise ValueError("reserved must be a bool (or uint8) mask [num_pages] on the pool's device")
    return mask.contiguous()


def copy_kv_pages(paged_kv_cache, src_pages, dst_pages):
    """Copy page ``src_pages[i]`` to page ``dst_pages[i]`` in every layer, in place.  No
    destination may be the source or destination of another copy."""
    dev = _lib.require_cuda(paged_kv_cache)
    pool = _pool(paged_kv_cache)
    src, dst = _i32(src_pages, dev), _i32(dst_pages, dev)
    if src.dim() != 1 or src.shape != dst.shape:
        raise ValueError("src_pages and dst_pages must be lists of the same length")
    with _lib.on_device(dev):
        _lib.check(_lib.lib().akt_copy_kv_pages(ctypes.byref(pool), src.data_ptr(), dst.data_ptr(), src.numel(),
                                                _lib.stream_ptr(dev)))
    return paged_kv_cache


def fork_paged_kv_cache(paged_kv_cache, kv_page_indptr, kv_page_indices, kv_last_page_len, parents, reserved=None,
                        max_entries=None):
    """A new batch of sequences: child ``c`` continues sequence ``parents[c]``.

    The first child of a parent takes its pages over; each further child shares the full
    pages and gets its own copy of a partly filled last page, in the lowest-numbered pages
    that neither a named parent nor ``reserved`` holds.  Sequences that no child names are
    dropped.  So beam search's reordering, several samples of one prompt and dropping
    finished sequences (``parents`` = those that stay) are all this call.

    parents: [num_children] (int32)
    max_entries: length of the returned index array (``sum`` of the children's pages; a
        longer one is -1 past its end).  None: computed, which costs one device-to-host read
    returns (kv_page_indptr [num_children + 1], kv_page_indices [max_entries],
        kv_last_page_len [num_children]), int32
    """
    dev = _lib.require_cuda(paged_kv_cache)
    a = _lib.ForkPagedArgs()
    a.pool = _pool(paged_kv_cache)
    indptr, indices, last = _i32(kv_page_indptr, dev), _i32(kv_page_indices, dev), _i32(kv_last_page_len, dev)
    par = _i32(parents, dev)
    B, F = indptr.numel() - 1, par.numel()
    if B < 0 or last.numel() != B or par.dim() != 1:
        raise ValueError("kv_page_indptr must have B+1 entries, kv_last_page_len B entries and parents be a list")
    mask = _reserved(reserved, a.pool.num_pages, dev)
    if max_entries is None:
        at = par.long().clamp(0, max(B - 1, 0))
        max_entries = int((indptr[at + 1] - indptr[at]).sum()) if B and F else 0
    if max_entries < 0:
        raise ValueError("max_entries must not be negative")
    i32 = dict(dtype=torch.int32, device=dev)
    out = (torch.empty(F + 1, **i32), torch.empty(max_entries, **i32), torch.empty(F, **i32))
    a.kv_page_indptr, a.kv_page_indices, a.kv_last_page_len = indptr.data_ptr(), indices.data_ptr(), last.data_ptr()
    a.num_page_entries = indices.numel()
    a.parents, a.reserved = par.data_ptr(), mask.data_ptr() if mask is not None else None
    a.out_indptr, a.out_indices, a.out_last_page_len = (t.data_ptr() for t in out)
    a.max_entries, a.batch, a.num_children = max_entries, B, F
    L = _lib.lib()
    with _lib.on_device(dev):
        ws = _lib.workspace(L.akt_fork_paged_workspace_size(ctypes.byref(a)), dev)
        _lib.check(L.akt_fork_paged(ctypes.byref(a), ws.data_ptr(), ws.numel(), _lib.stream_ptr(dev)))
    return out


def compact_paged_kv_cache(paged_kv_cache, kv_page_indices, reserved=None):
    """Move the live pages to the lowest page numbers that ``reserved`` leaves open, in
    place, so that the pool's tail is free.

    returns (kv_page_indices of the same length, pages_used): ``pages_used`` (int32 scalar
    on the device) is one past the highest page then in use or reserved.  ``kv_page_indptr``
    and ``kv_last_page_len`` stay as they are.
    """
    dev = _lib.require_cuda(paged_kv_cache)
    a = _lib.CompactPagedArgs()
    a.pool = _pool(paged_kv_cache)
    indices = _i32(kv_page_indices, dev)
    if indices.dim() != 1:
        raise ValueError("kv_page_indices must be a list")
    mask = _reserved(reserved, a.pool.num_pages, dev)
    out = torch.empty_like(indices)
    used = torch.empty((), dtype=torch.int32, device=dev)
    a.kv_page_indices, a.num_page_entries = indices.data_ptr(), indices.numel()
    a.reserved = mask.data_ptr() if mask is not None else None
    a.out_indices, a.pages_used = out.data_ptr(), used.data_ptr()
    L = _lib.lib()
    with _lib.on_device(dev):
        ws = _lib.workspace(L.akt_compact_paged_workspace_size(ctypes.byref(a)), dev)
        _lib.check(L.akt_compact_paged(ctypes.byref(a), ws.data_ptr(), ws.numel(), _lib.stream_ptr(dev)))
    return out, used


def free_kv_pages(num_pages, kv_page_indices, reserved=None):
    """The pages that the table does not name, ascending: ``(pages [num_pages] int32, -1 past
    their count; count, int32 scalar on the device)``."""
    dev = _lib.require_cuda(kv_page_indices)
    indices = _i32(kv_page_indices, dev)
    mask = _reserved(reserved, num_pages, dev)
    out = torch.empty(num_pages, dtype=torch.int32, device=dev)
    count = torch.empty((), dtype=torch.int32, device=dev)
    L = _lib.lib()
    with _lib.on_device(dev):
        ws = _lib.workspace(L.akt_free_kv_pages_workspace_size(num_pages), dev)
        _lib.check(L.akt_free_kv_pages(indices.data_ptr(), indices.numel(),
                                       mask.data_ptr() if mask is not None else None, num_pages, out.data_ptr(),
                                       count.data_ptr(), ws.data_ptr(), ws.numel(), _lib.stream_ptr(dev)))
    return out, count

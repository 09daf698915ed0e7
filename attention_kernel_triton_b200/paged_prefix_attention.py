"""Attention over a paged cache for a batch in which groups of sequences share
their first pages: the shared keys and values are read once for each group.

``fork_paged_kv_cache`` makes such batches (several samples of one prompt, beams,
conversations behind one system prompt): its children share their parent's full
pages.  The other attentions of the package read those once per sequence; here the
rows of all sequences of a group attend to the shared pages together, each row to its
own pages behind them, and the two results are joined by their log-sum-exps.  Queries,
pool, table, masks and results are those of
``paged_chunk_attention.flash_attention_chunk_paged`` (up to rounding); single tokens,
drafted tokens and prompt chunks alike.  The two results are kept in fp32 until they
are joined.  No gradient.  Runs ``akt_prefix_paged`` (sm_100a) on torch's current stream.

The workspace of a call with groups holds both fp32 results of every row, ``8 T Hq D``
bytes: chunks of long prompts are better small.

The sequences of a group stand side by side in the batch: group ``g`` is
``group_indptr[g]:group_indptr[g + 1]`` (a fork's ``parents`` in that order give it).
"""
from __future__ import annotations

import math

import torch

from . import _lib
from .paged_chunk_attention import _on_grid

_prefix = _lib.Entry("akt_prefix_paged", _lib.PrefixPagedArgs, _lib.c_void_p, _lib.c_size_t, _lib.c_void_p)
_workspace = _lib.Entry("akt_prefix_paged_workspace_size", _lib.PrefixPagedArgs, restype=_lib.c_size_t)


def shared_prefix_pages(group_indptr, kv_page_indptr, kv_page_indices, kv_last_page_len, page_size):
    """How many full pages all sequences of each group have in common from the first on
    (``[G]`` int32; 0 for fewer than two sequences).  It holds while the sequences only grow."""
    index = _lib.device_index(kv_page_indices)
    groups = _lib.list_i32(group_indptr, kv_page_indices)
    indptr, indices = _lib.list_i32(kv_page_indptr, kv_page_indices), _lib.list_i32(kv_page_indices, kv_page_indices)
    last = _lib.list_i32(kv_last_page_len, kv_page_indices)
    B, G = indptr.numel() - 1, groups.numel() - 1
    if B < 0 or G < 0 or last.numel() != B:
        raise ValueError("group_indptr must have G+1 entries, kv_page_indptr B+1 and kv_last_page_len B entries")
    out = indices.new_empty(G)
    with _lib.on_index(index):
        _lib.check(_lib.lib().akt_shared_prefix_pages(groups.data_ptr(), G, indptr.data_ptr(), indices.data_ptr(),
                                                      last.data_ptr(), B, indices.numel(), page_size, out.data_ptr(),
                                                      _lib.raw_stream(index)))
    return out


def shared_prefix_paged_into(out, q, q_indptr, paged_kv_cache, kv_page_indptr, kv_page_indices, kv_last_page_len,
                             group_indptr, shared_pages=None, causal=True, softmax_scale=None, lse=None):
    """Write the attention of ``q [T, Hq, D]`` into ``out [T, Hq, D]`` and, with ``lse`` (fp32
    ``[T, Hq]``), each row's natural-log sum-exp of the scaled scores (-inf where no key is seen)."""
    index = _lib.device_index(q, paged_kv_cache, out)
    if q.dtype != paged_kv_cache.dtype or out.dtype != q.dtype:
        raise TypeError("q, paged_kv_cache and the output must share one dtype")
    shape, pool = q.shape, paged_kv_cache.shape
    if len(shape) != 3 or out.shape != shape:
        raise ValueError("q and the output must be [T, Hq, D]")
    T, Hq, D = shape
    if len(pool) != 5 or pool[1] != 2 or pool[4] != D:
        raise ValueError("paged_kv_cache must be [num_pages, 2, Hkv, page_size, D]")
    lp = (0, 0, 0)
    if lse is not None:
        _lib.device_index(q, lse)
        if lse.dtype is not torch.float32 or lse.shape != shape[:2]:
            raise ValueError("lse must be fp32 [T, Hq]")
        lp = (lse.data_ptr(), *lse.stride())
    at, indptr = _lib.list_i32(q_indptr, q), _lib.list_i32(kv_page_indptr, q)
    indices, last = _lib.list_i32(kv_page_indices, q), _lib.list_i32(kv_last_page_len, q)
    groups = _lib.list_i32(group_indptr, q)
    B, G = indptr.numel() - 1, groups.numel() - 1
    if at.numel() != B + 1 or last.numel() != B:
        raise ValueError("q_indptr and kv_page_indptr must have B+1 entries and kv_last_page_len B entries")
    if shared_pages is None:
        shared_pages = shared_prefix_pages(groups, indptr, indices, last, pool[3])
    pages = _lib.list_i32(shared_pages, q)
    if G < 0 or pages.numel() != G:
        raise ValueError("group_indptr must have G+1 entries and shared_pages G entries")
    scale = 1.0 / math.sqrt(D) if softmax_scale is None else float(softmax_scale)
    tail = (indptr.data_ptr(), indices.data_ptr(), last.data_ptr(), indices.numel(), out.data_ptr(), *out.stride(), *lp,
            B, Hq, pool[2], pool[3], D, bool(causal), _lib.dtype_code(q), scale, groups.data_ptr(), pages.data_ptr(), G)

    def call(q, cache):
        values = (q.data_ptr(), *q.stride(), at.data_ptr(), T, cache.data_ptr(), *cache.stride(), pool[0], *tail)
        args = _prefix.pack(values)
        size = _workspace.packed(args)
        ws = q.new_empty((size + 1) // 2)
        return _prefix.packed(args, ws.data_ptr(), size, _lib.raw_stream(index))

    with _lib.on_index(index):
        rc = call(q, paged_kv_cache)
        if rc == _lib.AKT_ERR_UNSUPPORTED and D in (64, 128) and Hq <= 128 * pool[2] and _on_grid(out):
            # a layout: what is off the 16-byte grid is copied, then both (strides that no tensor map takes)
            q, cache = (t if _on_grid(t) else t.clone(memory_format=torch.contiguous_format) for t in (q, paged_kv_cache))
            rc = call(q, cache)
            if rc == _lib.AKT_ERR_UNSUPPORTED:
                rc = call(q.contiguous(), cache.contiguous())
        _lib.check(rc)
    return out


def flash_attention_shared_prefix_paged(q, q_indptr, paged_kv_cache, kv_page_indptr, kv_page_indices, kv_last_page_len,
                                        group_indptr, shared_pages=None, causal=True, softmax_scale=None):
    """
    q .. kv_last_page_len: those of ``flash_attention_chunk_paged``
    group_indptr: [G+1] (int32), bounds of the groups in the batch, ascending; a sequence
        outside all of them is one of its own
    shared_pages: [G] (int32), how many first pages the sequences of each group have in
        common; None: found by ``shared_prefix_pages``
    returns O: [T, Hq, D] in q.dtype; scale 1/sqrt(D) unless given
    """
    O = q.new_empty(q.shape)
    return shared_prefix_paged_into(O, q, q_indptr, paged_kv_cache, kv_page_indptr, kv_page_indices, kv_last_page_len,
                                    group_indptr, shared_pages, causal, softmax_scale)


def flash_attention_shared_prefix_paged_with_lse(q, q_indptr, paged_kv_cache, kv_page_indptr, kv_page_indices,
                                                 kv_last_page_len, group_indptr, shared_pages=None, causal=True,
                                                 softmax_scale=None):
    """``flash_attention_shared_prefix_paged`` returning ``(O, LSE)`` with fp32 ``LSE [T, Hq]``, the
    row's natural-log sum-exp of the scaled scores (-inf where no key is seen)."""
    O, lse = q.new_empty(q.shape), q.new_empty(q.shape[:2], dtype=torch.float32)
    shared_prefix_paged_into(O, q, q_indptr, paged_kv_cache, kv_page_indptr, kv_page_indices, kv_last_page_len,
                             group_indptr, shared_pages, causal, softmax_scale, lse)
    return O, lse

"""Attention of a chunk of new tokens over a paged cache: chunks of prompts,
drafted tokens to verify and single decoded tokens, ragged in one batch.

The reference has the one-token form
(``decode_flash_attention_redundant_var_len_paged.py:228-274``); the pool, the
page table and the scale are those of that module's
``flash_attention_decode_paged``.  Sequence ``b``'s queries are rows
``q_indptr[b]:q_indptr[b + 1]`` of ``q``, its ``n_b`` newest tokens, whose K and
V are in the pool already (``append_paged_kv_cache`` or
``append_rotary_paged_kv_cache`` with the same ``indptr``): row ``i`` stands at
position ``len_b - n_b + i``.  With ``causal`` it sees the keys up to its own
position, else all ``len_b``.  A row that sees no key (an empty sequence, a chunk
longer than its sequence) or that no sequence has gives zeros.  Scores, sums and
partial results are in fp32; the softmax weights are rounded to the inputs' type
for the product with V, as in the package's prefill and decode.  No gradient.
Runs ``akt_chunk_paged`` (sm_100a) on torch's current stream.
"""
from __future__ import annotations

import math

import torch

from . import _lib


_chunk = _lib.Entry("akt_chunk_paged", _lib.ChunkPagedArgs, _lib.c_void_p, _lib.c_size_t, _lib.c_void_p)
_workspace = _lib.Entry("akt_chunk_paged_workspace_size", _lib.ChunkPagedArgs, restype=_lib.c_size_t)


def chunk_paged_into(out, q, q_indptr, paged_kv_cache, kv_page_indptr, kv_page_indices, kv_last_page_len, causal=True,
                     softmax_scale=None, lse=None):
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
    B = indptr.numel() - 1
    if at.numel() != B + 1 or last.numel() != B:
        raise ValueError("q_indptr and kv_page_indptr must have B+1 entries and kv_last_page_len B entries")
    scale = 1.0 / math.sqrt(D) if softmax_scale is None else float(softmax_scale)
    tail = (indptr.data_ptr(), indices.data_ptr(), last.data_ptr(), indices.numel(), out.data_ptr(), *out.stride(), *lp,
            B, Hq, pool[2], pool[3], D, bool(causal), _lib.dtype_code(q), scale)

    def call(q, cache):
        values = (q.data_ptr(), *q.stride(), at.data_ptr(), T, cache.data_ptr(), *cache.stride(), pool[0], *tail)
        size = _workspace(values)
        ws = q.new_empty((size + 1) // 2)
        return _chunk(values, ws.data_ptr(), size, _lib.raw_stream(index))

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


def _on_grid(t):
    *strides, unit = t.stride()
    return unit == 1 and t.data_ptr() % 16 == 0 and all(s % 8 == 0 for s in strides)


def flash_attention_chunk_paged(q, q_indptr, paged_kv_cache, kv_page_indptr, kv_page_indices, kv_last_page_len,
                                causal=True, softmax_scale=None):
    """
    q: [T, Hq, D], the new tokens' queries of all sequences, ragged by q_indptr [B+1] (int32)
    paged_kv_cache: [all_num_pages, 2, Hkv, page_size, D] (2 for k and v; Hq a multiple of Hkv)
    kv_page_indptr: [B+1], kv_page_indices: [total_num_pages], kv_last_page_len: [B] (int32),
        the page table with the new tokens in it
    returns O: [T, Hq, D] in q.dtype; scale 1/sqrt(D) unless given
    """
    O = q.new_empty(q.shape)
    return chunk_paged_into(O, q, q_indptr, paged_kv_cache, kv_page_indptr, kv_page_indices, kv_last_page_len, causal,
                            softmax_scale)


def flash_attention_chunk_paged_with_lse(q, q_indptr, paged_kv_cache, kv_page_indptr, kv_page_indices,
                                         kv_last_page_len, causal=True, softmax_scale=None):
    """``flash_attention_chunk_paged`` returning ``(O, LSE)`` with fp32 ``LSE [T, Hq]``, the
    row's natural-log sum-exp of the scaled scores (-inf where no key is seen), which merges
    with other partial results (``akt_lse_merge``)."""
    O, lse = q.new_empty(q.shape), q.new_empty(q.shape[:2], dtype=torch.float32)
    chunk_paged_into(O, q, q_indptr, paged_kv_cache, kv_page_indptr, kv_page_indices, kv_last_page_len, causal,
                     softmax_scale, lse)
    return O, lse

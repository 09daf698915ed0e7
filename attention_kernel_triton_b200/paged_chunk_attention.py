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
longer than its sequence) gives zeros.  Runs ``akt_chunk_paged`` (sm_100a) on
torch's current stream.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib


def _i32(t, dev):
    return _lib.as_int32(t, dev).contiguous()


def chunk_paged_into(out, q, q_indptr, paged_kv_cache, kv_page_indptr, kv_page_indices, kv_last_page_len, causal=True,
                     softmax_scale=None, lse=None):
    """Write the attention of ``q [T, Hq, D]`` into ``out [T, Hq, D]`` and, with ``lse`` (fp32
    ``[T, Hq]``), each row's natural-log sum-exp of the scaled scores (-inf where no key is seen)."""
    dev = _lib.require_cuda(q, paged_kv_cache, out)
    if q.dtype != paged_kv_cache.dtype or out.dtype != q.dtype:
        raise TypeError("q, paged_kv_cache and the output must share one dtype")
    if q.dim() != 3 or out.shape != q.shape:
        raise ValueError("q and the output must be [T, Hq, D]")
    T, Hq, D = q.shape
    if paged_kv_cache.dim() != 5 or paged_kv_cache.shape[1] != 2 or paged_kv_cache.shape[4] != D:
        raise ValueError("paged_kv_cache must be [num_pages, 2, Hkv, page_size, D]")
    if lse is not None:
        _lib.require_cuda(q, lse)
        if lse.dtype != torch.float32 or lse.shape != (T, Hq):
            raise ValueError("lse must be fp32 [T, Hq]")
    at, indptr = _i32(q_indptr, dev), _i32(kv_page_indptr, dev)
    indices, last = _i32(kv_page_indices, dev), _i32(kv_last_page_len, dev)
    B = indptr.numel() - 1
    if at.numel() != B + 1 or last.numel() != B:
        raise ValueError("q_indptr and kv_page_indptr must have B+1 entries and kv_last_page_len B entries")
    t = {"q": q, "cache": paged_kv_cache}
    a = _lib.ChunkPagedArgs()
    a.q_indptr, a.num_tokens = at.data_ptr(), T
    a.kv_page_indptr, a.kv_page_indices, a.kv_last_page_len = indptr.data_ptr(), indices.data_ptr(), last.data_ptr()
    a.num_page_entries = indices.numel()
    a.out, (a.out_stride_token, a.out_stride_head, a.out_stride_dim) = out.data_ptr(), out.stride()
    if lse is not None:
        a.lse, (a.lse_stride_token, a.lse_stride_head) = lse.data_ptr(), lse.stride()
    a.batch, a.num_qo_heads, a.num_kv_heads = B, Hq, paged_kv_cache.shape[2]
    a.page_size, a.head_dim, a.causal = paged_kv_cache.shape[3], D, int(bool(causal))
    a.dtype = _lib.dtype_code(q)
    a.softmax_scale = 1.0 / math.sqrt(D) if softmax_scale is None else float(softmax_scale)
    L = _lib.lib()

    def call():
        qq, cache = t["q"], t["cache"]
        a.q, (a.q_stride_token, a.q_stride_head, a.q_stride_dim) = qq.data_ptr(), qq.stride()
        a.kv_cache, a.num_pages = cache.data_ptr(), cache.shape[0]
        (a.kv_stride_page, a.kv_stride_kv, a.kv_stride_head, a.kv_stride_token, a.kv_stride_dim) = cache.stride()
        ws = _lib.workspace(L.akt_chunk_paged_workspace_size(ctypes.byref(a)), dev)
        return L.akt_chunk_paged(ctypes.byref(a), ws.data_ptr(), ws.numel(), _lib.stream_ptr(dev))

    def contiguous():
        for k in t:
            t[k] = t[k].contiguous()

    with _lib.on_device(dev):
        _lib.run_with_layout_retry(call, contiguous)
    return out


def flash_attention_chunk_paged(q, q_indptr, paged_kv_cache, kv_page_indptr, kv_page_indices, kv_last_page_len,
                                causal=True, softmax_scale=None):
    """
    q: [T, Hq, D], the new tokens' queries of all sequences, ragged by q_indptr [B+1] (int32)
    paged_kv_cache: [all_num_pages, 2, Hkv, page_size, D] (2 for k and v; Hq a multiple of Hkv)
    kv_page_indptr: [B+1], kv_page_indices: [total_num_pages], kv_last_page_len: [B] (int32),
        the page table with the new tokens in it
    returns O: [T, Hq, D] in q.dtype; scale 1/sqrt(D) unless given
    """
    O = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    return chunk_paged_into(O, q, q_indptr, paged_kv_cache, kv_page_indptr, kv_page_indices, kv_last_page_len, causal,
                            softmax_scale)


def flash_attention_chunk_paged_with_lse(q, q_indptr, paged_kv_cache, kv_page_indptr, kv_page_indices,
                                         kv_last_page_len, causal=True, softmax_scale=None):
    """``flash_attention_chunk_paged`` returning ``(O, LSE)`` with fp32 ``LSE [T, Hq]``, the
    row's natural-log sum-exp of the scaled scores (-inf where no key is seen), which merges
    with other partial results (``akt_lse_merge``)."""
    O = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
    chunk_paged_into(O, q, q_indptr, paged_kv_cache, kv_page_indptr, kv_page_indices, kv_last_page_len, causal,
                     softmax_scale, lse)
    return O, lse

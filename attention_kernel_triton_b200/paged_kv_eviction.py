"""Eviction from a paged KV cache by accumulated attention weight: what weight
each key has got, which tokens of each head stay, and the pool with only those.

The reference's sparse decodes take lists of kept tokens per head
(``sparsetoken_decode_flash_attention_redundant_var_len_paged.py``); nothing in
it chooses them or shrinks a cache.  Three steps, on torch's current stream
(sm_100a, ``csrc/weights.cu``, ``csrc/evict.cu``):

1. ``accumulate_attention_weights_paged`` after an attention that returned its
   log-sum-exp (``flash_attention_chunk_paged_with_lse`` or
   ``flash_attention_shared_prefix_paged_with_lse``): the softmax weight of each key,
   summed over the new queries and the query heads of its kv head, added to a
   ``weights [B, Hkv, L]`` array (fp32; key ``j`` of sequence ``b`` is ``[b, :, j]``)
   that the caller keeps beside the pool.
2. ``select_kept_tokens``: per head the first tokens, the newest ones and the
   heaviest of the rest, as lists in the format of the package's sparse decodes
   (``sparse_ind``), which can attend to them without any eviction.
3. ``evict_paged_kv_cache``: the kept rows moved to the front of their sequence, a
   new page table, the weights moved along.

Each head keeps its own tokens, so after an eviction slot ``i`` of two heads may be
different tokens: keys must be in the pool with their positions applied
(``append_rotary_paged_kv_cache`` or ``apply_rotary_qk`` before the append), and the
positions of later tokens are the caller's to count (the table's lengths no longer give
them: ``apply_rotary_qk`` with ``positions``, then ``append_paged_kv_cache``).
No gradient.
"""
from __future__ import annotations

import math

import torch

from . import _lib
from .paged_chunk_attention import _on_grid
from .paged_kv_pages import _pool, _ptr, _reserved

_weights = _lib.Entry("akt_attention_weights", _lib.AttentionWeightsArgs, _lib.c_void_p, _lib.c_size_t, _lib.c_void_p)
_weights_size = _lib.Entry("akt_attention_weights_workspace_size", _lib.AttentionWeightsArgs, restype=_lib.c_size_t)
_select = _lib.Entry("akt_select_tokens", _lib.SelectTokensArgs, _lib.c_void_p)
_evict = _lib.Entry("akt_evict_paged", _lib.EvictPagedArgs, _lib.c_void_p, _lib.c_size_t, _lib.c_void_p)
_evict_size = _lib.Entry("akt_evict_paged_workspace_size", _lib.EvictPagedArgs, restype=_lib.c_size_t)


def _unit(t):
    """Whether the last dimension's values stand side by side."""
    return t.stride(-1) == 1 or t.shape[-1] <= 1


def accumulate_attention_weights_paged(weights, q, q_indptr, paged_kv_cache, kv_page_indptr, kv_page_indices,
                                       kv_last_page_len, lse, causal=True, softmax_scale=None, out=None):
    """Add to ``weights[b, h, j]`` the softmax weights that key ``j`` of sequence ``b`` gets
    from the queries of kv head ``h``'s query heads: the sum of ``exp(scale q . k_j - lse)``
    over the rows of ``q`` that see it.

    weights: [B, Hkv, L] fp32, L no less than the longest sequence; None: from zero, into ``out``
    q .. softmax_scale: those of ``flash_attention_chunk_paged_with_lse``, whose second result is
    lse: [T, Hq] fp32, over all keys that the row sees (with another one the sums are not of
        softmax weights, and may pass fp32's range); a row of -inf adds nothing
    out: [B, Hkv, L] fp32 for the sums; None: ``weights`` itself
    returns out; its places past a sequence's length stay as they were
    """
    out = weights if out is None else out
    if out is None:
        raise ValueError("weights or out must be given")
    index = _lib.device_index(q, paged_kv_cache, lse, out)
    if q.dtype != paged_kv_cache.dtype:
        raise TypeError("q and paged_kv_cache must share one dtype")
    shape, pool = q.shape, paged_kv_cache.shape
    if len(shape) != 3:
        raise ValueError("q must be [T, Hq, D]")
    T, Hq, D = shape
    if len(pool) != 5 or pool[1] != 2 or pool[4] != D:
        raise ValueError("paged_kv_cache must be [num_pages, 2, Hkv, page_size, D]")
    if lse.dtype is not torch.float32 or lse.shape != shape[:2]:
        raise ValueError("lse must be fp32 [T, Hq]")
    at, indptr = _lib.list_i32(q_indptr, q), _lib.list_i32(kv_page_indptr, q)
    indices, last = _lib.list_i32(kv_page_indices, q), _lib.list_i32(kv_last_page_len, q)
    B = indptr.numel() - 1
    if at.numel() != B + 1 or last.numel() != B:
        raise ValueError("q_indptr and kv_page_indptr must have B+1 entries and kv_last_page_len B entries")
    for t in (out,) if weights is None or weights is out else (out, weights):
        if t.dtype is not torch.float32 or len(t.shape) != 3 or t.shape[:2] != (B, pool[2]) or t.shape != out.shape:
            raise ValueError("weights and out must be fp32 [B, Hkv, L]")
        if not _unit(t):
            raise ValueError("weights and out must have unit stride in their last dimension")
    if weights is None:
        start = (0, 0, 0)
    else:
        _lib.device_index(q, weights)
        start = (weights.data_ptr(), *weights.stride()[:2])
    scale = 1.0 / math.sqrt(D) if softmax_scale is None else float(softmax_scale)
    tail = (indptr.data_ptr(), indices.data_ptr(), last.data_ptr(), indices.numel(), lse.data_ptr(), *lse.stride(),
            *start, out.data_ptr(), *out.stride()[:2], out.shape[2], B, Hq, pool[2], pool[3], D, bool(causal),
            _lib.dtype_code(q), scale)

    def call(q, cache):
        values = (q.data_ptr(), *q.stride(), at.data_ptr(), T, cache.data_ptr(), *cache.stride(), pool[0], *tail)
        args = _weights.pack(values)
        size = _weights_size.packed(args)
        ws = q.new_empty((size + 1) // 2)
        return _weights.packed(args, ws.data_ptr(), size, _lib.raw_stream(index))

    with _lib.on_index(index):
        rc = call(q, paged_kv_cache)
        if rc == _lib.AKT_ERR_UNSUPPORTED and D in (64, 128) and Hq <= 128 * pool[2]:
            # a layout: what is off the 16-byte grid is copied, then both (strides that no tensor map takes)
            q, cache = (t if _on_grid(t) else t.clone(memory_format=torch.contiguous_format) for t in (q, paged_kv_cache))
            rc = call(q, cache)
            if rc == _lib.AKT_ERR_UNSUPPORTED:
                rc = call(q.contiguous(), cache.contiguous())
        _lib.check(rc)
    return out


def select_kept_tokens(weights, seq_lens, budget, sinks=0, recent=0):
    """Which ``min(seq_lens[b], budget)`` tokens of each head stay: the first ``sinks``, the
    last ``recent`` and the heaviest of the others (the lowest index of equal weights; NaN
    counts as below everything).

    weights: [B, H, L] fp32, or [layers, B, H, L] with lists for each layer
    seq_lens: [B] (int32), tokens of each sequence
    returns (keep_ind [(layers,) B, H, budget] int32, ascending, 0 past the kept ones;
        keep_len [B] int32)
    """
    index = _lib.device_index(weights)
    shape = weights.shape
    if weights.dtype is not torch.float32 or len(shape) not in (3, 4):
        raise ValueError("weights must be fp32 [B, H, L] or [layers, B, H, L]")
    if budget < 0 or sinks < 0 or recent < 0 or sinks + recent > budget:
        raise ValueError("budget, sinks and recent must not be negative, and sinks + recent at most the budget")
    lens = _lib.list_i32(seq_lens, weights)
    *layers, B, H, L = shape
    if lens.dim() != 1 or lens.shape[0] != B:
        raise ValueError("seq_lens must have B entries")
    w = weights if _unit(weights) else weights.contiguous()
    ind, kept = lens.new_empty((*layers, B, H, budget)), lens.new_empty(B)
    ws, si = w.stride(), ind.stride()
    ws, si = (ws[-4] if layers else 0, *ws[-3:-1]), (si[-4] if layers else 0, *si[-3:-1])
    with _lib.on_index(index):
        rc = _select((w.data_ptr(), *ws, lens.data_ptr(), ind.data_ptr(), *si, kept.data_ptr(), L,
                      layers[0] if layers else 1, B, H, budget, sinks, recent), _lib.raw_stream(index))
        if rc:
            _lib.check(rc)
    return ind, kept


def evict_paged_kv_cache(paged_kv_cache, kv_page_indptr, kv_page_indices, kv_last_page_len, keep_ind, keep_len,
                         weights=None, reserved=None):
    """Move the kept tokens of each head to the front of their sequence, in place: slot ``i``
    of head ``h`` takes the row of token ``keep_ind[b, h, i]``, for ``i < keep_len[b]``.

    A sequence stays in its first pages.  No page that another entry of the table names too
    (a forked prefix) or that ``reserved`` marks is written: one that is full of rows that
    stay in place is shared further, any other is replaced by the lowest-numbered dead page
    (-1 and lost rows where there is none; ``_lib.device_status`` tells).  The table must
    be the whole pool's.  The pages behind the new table's are then dead.

    paged_kv_cache: [num_pages, 2, Hkv, page_size, D], or with layers before it
    keep_ind: [(layers,) B, Hkv, M] (int32), ascending in each list; keep_len: [B] (int32)
    weights: [(layers,) B, Hkv, L] fp32 or None: moved along in place, zeros in the places left
    returns (kv_page_indptr [B + 1], kv_page_indices, kv_last_page_len [B]), int32; the index
        array is as long as the lists can need (-1 past its end)
    """
    index = _lib.device_index(paged_kv_cache)
    pool = _pool(paged_kv_cache)
    indptr, indices = _lib.list_i32(kv_page_indptr, paged_kv_cache), _lib.list_i32(kv_page_indices, paged_kv_cache)
    last, kept = _lib.list_i32(kv_last_page_len, paged_kv_cache), _lib.list_i32(keep_len, paged_kv_cache)
    keep = keep_ind
    if keep.dtype is not torch.int32 or keep.get_device() != index:
        keep = keep.to(device=paged_kv_cache.device, dtype=torch.int32)
    layered, B = len(paged_kv_cache.shape) == 6, indptr.numel() - 1
    heads = (*paged_kv_cache.shape[:1], B, pool[9]) if layered else (B, pool[9])
    if B < 0 or last.numel() != B or kept.numel() != B:
        raise ValueError("kv_page_indptr must have B+1 entries, kv_last_page_len and keep_len B entries")
    if keep.shape[:-1] != heads or len(keep.shape) != len(heads) + 1:
        raise ValueError("keep_ind must be [B, Hkv, M], with the pool's layers before it or not")
    keep = keep if _unit(keep) else keep.contiguous()
    ks, M = keep.stride(), keep.shape[-1]
    wp = (0, 0, 0, 0, 0)
    if weights is not None:
        _lib.device_index(paged_kv_cache, weights)
        if weights.dtype is not torch.float32 or weights.shape[:-1] != heads or len(weights.shape) != len(heads) + 1:
            raise ValueError("weights must be fp32 [B, Hkv, L], with the pool's layers before it or not")
        if not _unit(weights):
            raise ValueError("weights must have unit stride in their last dimension")
        st = weights.stride()
        wp = (weights.data_ptr(), st[0] if layered else 0, *st[-3:-1], weights.shape[-1])
    mask = _reserved(reserved, pool[7], paged_kv_cache)
    most = min(B * -(-M // pool[10]), indices.numel())
    # the new table in one allocation; the workspace has its own, which goes when the call ends
    out_indptr, out_indices, out_last = indptr.new_empty(2 * B + 1 + most).split_with_sizes((B + 1, most, B))
    values = (*pool, indptr.data_ptr(), indices.data_ptr(), last.data_ptr(), indices.numel(), keep.data_ptr(),
              ks[0] if layered else 0, *ks[-3:-1], kept.data_ptr(), M, _ptr(mask), *wp, out_indptr.data_ptr(),
              out_indices.data_ptr(), out_last.data_ptr(), most, B)
    args = _evict.pack(values)
    size = _evict_size.packed(args)
    ws = indptr.new_empty(size // 4 + 1)
    with _lib.on_index(index):
        rc = _evict.packed(args, ws.data_ptr(), size, _lib.raw_stream(index))
        if rc:
            _lib.check(rc)
    return out_indptr, out_indices, out_last

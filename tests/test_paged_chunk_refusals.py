"""What the chunk attention refuses, without a GPU."""
import ctypes

import pytest
import torch

from attention_kernel_triton_b200 import _lib
from attention_kernel_triton_b200.paged_chunk_attention import flash_attention_chunk_paged


def test_cpu_tensors_are_refused():
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        flash_attention_chunk_paged(torch.zeros(1, 2, 64), i, torch.zeros(1, 2, 1, 4, 64), i, i, i[:1])


def test_c_entry_refuses_bad_arguments():
    L = _lib.lib()

    def args(**kw):
        a = _lib.ChunkPagedArgs()
        a.batch, a.num_tokens, a.num_qo_heads, a.num_kv_heads, a.page_size, a.head_dim = 1, 4, 8, 2, 16, 128
        a.softmax_scale, a.num_pages, a.num_page_entries = 0.1, 3, 2
        a.q = a.out = a.kv_cache = a.q_indptr = a.kv_page_indptr = a.kv_page_indices = a.kv_last_page_len = 256
        a.q_stride_dim = a.kv_stride_dim = a.out_stride_dim = 1
        for k, v in kw.items():
            setattr(a, k, v)
        return a

    def rc(**kw):
        return L.akt_chunk_paged(ctypes.byref(args(**kw)), None, 0, None)

    for kw in (dict(num_qo_heads=7), dict(num_kv_heads=0), dict(page_size=0), dict(batch=-1), dict(num_tokens=-1),
               dict(softmax_scale=0.0), dict(softmax_scale=float("inf")), dict(softmax_scale=float("nan")), dict(dtype=7),
               dict(q=None), dict(q_indptr=None), dict(kv_page_indices=None), dict(batch=0), dict(num_tokens=1 << 40)):
        assert rc(**kw) == _lib.AKT_ERR_INVALID, kw
    for kw in (dict(head_dim=96), dict(q_stride_dim=2), dict(kv_stride_dim=128), dict(out_stride_dim=0)):
        assert rc(**kw) == _lib.AKT_ERR_UNSUPPORTED, kw
    assert rc(num_tokens=0) == _lib.AKT_OK
    assert L.akt_chunk_paged(None, None, 0, None) == _lib.AKT_ERR_INVALID

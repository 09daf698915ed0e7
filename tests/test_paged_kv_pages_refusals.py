"""What the page operators refuse, without a GPU."""
import ctypes

import pytest
import torch

from attention_kernel_triton_b200 import _lib
from attention_kernel_triton_b200.paged_kv_pages import (compact_paged_kv_cache, copy_kv_pages, fork_paged_kv_cache,
                                                         free_kv_pages)


def test_cpu_tensors_are_refused():
    pool = torch.zeros(2, 2, 1, 4, 8, dtype=torch.float16)
    i = torch.zeros(1, dtype=torch.int32)
    for call in (lambda: copy_kv_pages(pool, i, i), lambda: fork_paged_kv_cache(pool, i, i, i, i),
                 lambda: compact_paged_kv_cache(pool, i), lambda: free_kv_pages(2, i)):
        with pytest.raises(ValueError):
            call()


def test_c_entries_refuse_bad_arguments():
    L = _lib.lib()
    pool = _lib.PagePool()
    pool.kv_cache, pool.stride_dim, pool.num_pages = 16, 1, 4
    pool.num_layers = pool.num_kv_heads = pool.page_size = 1
    assert L.akt_copy_kv_pages(ctypes.byref(pool), None, None, 0, None) == _lib.AKT_ERR_INVALID  # head_dim 0
    pool.head_dim = 8
    assert L.akt_copy_kv_pages(ctypes.byref(pool), None, None, 0, None) == _lib.AKT_OK
    assert L.akt_copy_kv_pages(ctypes.byref(pool), None, None, 3, None) == _lib.AKT_ERR_INVALID
    assert L.akt_copy_kv_pages(ctypes.byref(pool), None, None, -1, None) == _lib.AKT_ERR_INVALID
    pool.stride_dim = 2
    assert L.akt_copy_kv_pages(ctypes.byref(pool), 16, 16, 1, None) == _lib.AKT_ERR_UNSUPPORTED
    pool.stride_dim = 1
    f = _lib.ForkPagedArgs()
    f.pool = pool
    f.batch, f.num_children, f.max_entries = 2, 3, 10
    assert L.akt_fork_paged(ctypes.byref(f), None, 0, None) == _lib.AKT_ERR_INVALID
    f.out_indptr = f.out_indices = f.out_last_page_len = f.parents = f.kv_page_indptr = f.kv_last_page_len = 16
    assert L.akt_fork_paged_workspace_size(ctypes.byref(f)) > 0
    assert L.akt_fork_paged(ctypes.byref(f), None, 0, None) == _lib.AKT_ERR_WORKSPACE
    f.num_children = -1
    assert L.akt_fork_paged(ctypes.byref(f), None, 0, None) == _lib.AKT_ERR_INVALID
    c = _lib.CompactPagedArgs()
    c.pool = pool
    assert L.akt_compact_paged(ctypes.byref(c), None, 0, None) == _lib.AKT_ERR_INVALID
    c.pages_used = 16
    assert L.akt_compact_paged(ctypes.byref(c), None, 0, None) == _lib.AKT_ERR_WORKSPACE
    assert L.akt_free_kv_pages(None, 3, None, 4, 16, 16, None, 0, None) == _lib.AKT_ERR_INVALID
    assert L.akt_free_kv_pages(None, 0, None, 1 << 30, 16, 16, None, 0, None) == _lib.AKT_ERR_WORKSPACE
    for fn in (L.akt_fork_paged, L.akt_compact_paged):
        assert fn(None, None, 0, None) == _lib.AKT_ERR_INVALID

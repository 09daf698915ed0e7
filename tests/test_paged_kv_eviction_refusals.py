"""What the eviction's entry points refuse, without a GPU, and their argument structs against the C layout."""
import ctypes
import os
import subprocess

import pytest
import torch

from attention_kernel_triton_b200 import _lib
from attention_kernel_triton_b200.paged_kv_eviction import (accumulate_attention_weights_paged, evict_paged_kv_cache,
                                                            select_kept_tokens)

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTS = {
    "akt_attention_weights_args": _lib.AttentionWeightsArgs,
    "akt_select_tokens_args": _lib.SelectTokensArgs,
    "akt_evict_paged_args": _lib.EvictPagedArgs,
}


def test_ctypes_structs_match_c_layout(tmp_path):
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "akt.h"', "int main(void){"]
    for cname, py in STRUCTS.items():
        lines.append(f'printf("{cname} size %zu\\n", sizeof({cname}));')
        for fname, _ in py._fields_:
            lines.append(f'printf("{cname} {fname} %zu\\n", offsetof({cname}, {fname}));')
    lines.append("return 0;}")
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split("\n")
    seen = 0
    for line in filter(None, out):
        cname, field, val = line.split()
        py = STRUCTS[cname]
        assert (ctypes.sizeof(py) if field == "size" else getattr(py, field).offset) == int(val), (cname, field)
        seen += 1
    assert seen == sum(len(s._fields_) + 1 for s in STRUCTS.values())


def test_cpu_tensors_are_refused():
    i, w = torch.zeros(2, dtype=torch.int32), torch.zeros(1, 1, 8)
    pool = torch.zeros(1, 2, 1, 4, 64)
    with pytest.raises(ValueError):
        accumulate_attention_weights_paged(w, torch.zeros(1, 2, 64), i, pool, i, i, i[:1], torch.zeros(1, 2))
    with pytest.raises(ValueError):
        accumulate_attention_weights_paged(None, torch.zeros(1, 2, 64), i, pool, i, i, i[:1], torch.zeros(1, 2))
    with pytest.raises(ValueError):
        select_kept_tokens(w, i[:1], 4)
    with pytest.raises(ValueError):
        evict_paged_kv_cache(pool.half(), i, i, i[:1], torch.zeros(1, 1, 4, dtype=torch.int32), i[:1])


def test_weights_entry_refuses_bad_arguments():
    L = _lib.lib()

    def rc(**kw):
        a = _lib.AttentionWeightsArgs()
        a.batch, a.num_tokens, a.num_qo_heads, a.num_kv_heads, a.page_size, a.head_dim = 1, 4, 8, 2, 16, 128
        a.softmax_scale, a.num_pages, a.num_page_entries, a.width = 0.1, 3, 2, 32
        a.q = a.out = a.lse = a.kv_cache = a.q_indptr = a.kv_page_indptr = a.kv_page_indices = a.kv_last_page_len = 256
        a.q_stride_dim = a.kv_stride_dim = 1
        for k, v in kw.items():
            setattr(a, k, v)
        return L.akt_attention_weights(ctypes.byref(a), None, 0, None)

    for kw in (dict(num_qo_heads=7), dict(num_kv_heads=0), dict(page_size=0), dict(batch=-1), dict(num_tokens=-1),
               dict(softmax_scale=0.0), dict(softmax_scale=float("inf")), dict(softmax_scale=float("nan")), dict(dtype=7),
               dict(q=None), dict(lse=None), dict(out=None), dict(q_indptr=None), dict(kv_page_indices=None),
               dict(num_tokens=1 << 40), dict(width=-1), dict(width=1 << 40)):
        assert rc(**kw) == _lib.AKT_ERR_INVALID, kw
    for kw in (dict(head_dim=96), dict(q_stride_dim=2), dict(kv_stride_dim=128), dict(q=264), dict(kv_stride_page=4),
               dict(num_qo_heads=258)):
        assert rc(**kw) == _lib.AKT_ERR_UNSUPPORTED, kw
    assert rc(batch=0) == _lib.AKT_OK
    assert L.akt_attention_weights(None, None, 0, None) == _lib.AKT_ERR_INVALID


def test_select_entry_refuses_bad_arguments():
    L = _lib.lib()

    def rc(**kw):
        a = _lib.SelectTokensArgs()
        a.layers, a.batch, a.num_heads, a.width, a.budget, a.sinks, a.recent = 1, 2, 2, 100, 10, 1, 2
        a.weights = a.seq_lens = a.keep_ind = a.keep_len = 256
        for k, v in kw.items():
            setattr(a, k, v)
        return L.akt_select_tokens(ctypes.byref(a), None)

    for kw in (dict(batch=-1), dict(layers=-1), dict(num_heads=-1), dict(width=-1), dict(budget=-1), dict(sinks=9),
               dict(recent=10), dict(sinks=-1), dict(weights=None), dict(seq_lens=None), dict(keep_ind=None),
               dict(keep_len=None), dict(num_heads=0), dict(layers=0), dict(width=1 << 40),
               dict(sinks=1 << 30, recent=1 << 30, budget=100)):
        assert rc(**kw) == _lib.AKT_ERR_INVALID, kw
    assert rc(batch=0) == _lib.AKT_OK
    assert L.akt_select_tokens(None, None) == _lib.AKT_ERR_INVALID


def test_evict_entry_refuses_bad_arguments():
    L = _lib.lib()

    def args(**kw):
        a = _lib.EvictPagedArgs()
        a.pool.kv_cache, a.pool.stride_dim, a.pool.num_pages = 16, 1, 4
        a.pool.num_layers = a.pool.num_kv_heads = a.pool.page_size = 1
        a.pool.head_dim = 8
        a.batch, a.num_page_entries, a.max_entries, a.max_kept = 2, 4, 4, 3
        a.kv_page_indptr = a.kv_page_indices = a.kv_last_page_len = a.keep_ind = a.keep_len = 256
        a.out_indptr = a.out_indices = a.out_last_page_len = 256
        for k, v in kw.items():
            setattr(a.pool if hasattr(a.pool, k) else a, k, v)
        return a

    def rc(**kw):
        return L.akt_evict_paged(ctypes.byref(args(**kw)), None, 0, None)

    for kw in (dict(num_layers=0), dict(page_size=0), dict(head_dim=0), dict(num_pages=-1), dict(batch=-1),
               dict(num_page_entries=-1), dict(max_entries=-1), dict(max_kept=-1), dict(width=-1), dict(kv_cache=None),
               dict(out_indptr=None), dict(out_indices=None), dict(out_last_page_len=None), dict(keep_ind=None),
               dict(keep_len=None), dict(kv_page_indptr=None), dict(kv_page_indices=None), dict(kv_last_page_len=None),
               dict(num_page_entries=1 << 40)):
        assert rc(**kw) == _lib.AKT_ERR_INVALID, kw
    assert rc(stride_dim=2) == _lib.AKT_ERR_UNSUPPORTED
    assert rc(head_dim=1 << 20) == _lib.AKT_ERR_UNSUPPORTED
    assert L.akt_evict_paged_workspace_size(ctypes.byref(args())) > 0
    assert rc() == _lib.AKT_ERR_WORKSPACE
    assert L.akt_evict_paged(None, None, 0, None) == _lib.AKT_ERR_INVALID

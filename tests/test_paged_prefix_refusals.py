"""What the attention behind shared prefixes refuses, without a GPU, and its argument struct against the C layout."""
import ctypes
import os
import subprocess

import pytest
import torch

from attention_kernel_triton_b200 import _lib
from attention_kernel_triton_b200.paged_prefix_attention import flash_attention_shared_prefix_paged, shared_prefix_pages

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_ctypes_struct_matches_c_layout(tmp_path):
    fields = [f for f, _ in _lib.PrefixPagedArgs._fields_]
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "akt.h"', "int main(void){",
             'printf("%zu\\n", sizeof(akt_prefix_paged_args));']
    lines += [f'printf("%zu\\n", offsetof(akt_prefix_paged_args, {f}));' for f in fields] + ["return 0;}"]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines))
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()
    want = [ctypes.sizeof(_lib.PrefixPagedArgs)] + [getattr(_lib.PrefixPagedArgs, f).offset for f in fields]
    assert [int(x) for x in out] == want


def test_cpu_tensors_are_refused():
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        flash_attention_shared_prefix_paged(torch.zeros(1, 2, 64), i, torch.zeros(1, 2, 1, 4, 64), i, i, i[:1], i, i[:1])
    with pytest.raises(ValueError):
        shared_prefix_pages(i, i, i, i[:1], 4)


def test_c_entries_refuse_bad_arguments():
    L = _lib.lib()

    def rc(**kw):
        a = _lib.PrefixPagedArgs()
        c = a.chunk
        c.batch, c.num_tokens, c.num_qo_heads, c.num_kv_heads, c.page_size, c.head_dim = 1, 4, 8, 2, 16, 128
        c.softmax_scale, c.num_pages, c.num_page_entries = 0.1, 3, 2
        c.q = c.out = c.kv_cache = c.q_indptr = c.kv_page_indptr = c.kv_page_indices = c.kv_last_page_len = 256
        c.q_stride_dim = c.kv_stride_dim = c.out_stride_dim = 1
        a.group_indptr = a.shared_pages = 256
        a.num_groups = 1
        for k, v in kw.items():
            setattr(c if hasattr(c, k) else a, k, v)
        return L.akt_prefix_paged(ctypes.byref(a), None, 0, None)

    for kw in (dict(num_groups=-1), dict(group_indptr=None), dict(shared_pages=None), dict(num_qo_heads=7), dict(batch=-1),
               dict(num_tokens=-1), dict(softmax_scale=0.0), dict(dtype=7), dict(q=None), dict(batch=0)):
        assert rc(**kw) == _lib.AKT_ERR_INVALID, kw
    for kw in (dict(head_dim=96), dict(q_stride_dim=2), dict(kv_stride_dim=128)):
        assert rc(**kw) == _lib.AKT_ERR_UNSUPPORTED, kw
    assert rc(num_tokens=0) == _lib.AKT_OK
    assert rc() == _lib.AKT_ERR_WORKSPACE
    assert L.akt_prefix_paged(None, None, 0, None) == _lib.AKT_ERR_INVALID
    p = 256
    assert L.akt_shared_prefix_pages(p, -1, p, p, p, 1, 1, 16, p, None) == _lib.AKT_ERR_INVALID
    assert L.akt_shared_prefix_pages(p, 1, p, p, p, 1, 1, 0, p, None) == _lib.AKT_ERR_INVALID
    assert L.akt_shared_prefix_pages(None, 1, p, p, p, 1, 1, 16, p, None) == _lib.AKT_ERR_INVALID
    assert L.akt_shared_prefix_pages(p, 1, p, None, p, 1, 1, 16, p, None) == _lib.AKT_ERR_INVALID
    assert L.akt_shared_prefix_pages(p, 0, p, p, p, 1, 1, 16, p, None) == _lib.AKT_OK

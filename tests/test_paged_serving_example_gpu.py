"""The serving example end to end, and the operators over a pool whose offsets pass 32 bits."""
import importlib.util
import os

import pytest
import torch

from attention_kernel_triton_b200 import _lib
from attention_kernel_triton_b200.paged_chunk_attention import flash_attention_chunk_paged
from attention_kernel_triton_b200.paged_kv_pages import compact_paged_kv_cache, copy_kv_pages, fork_paged_kv_cache
from attention_kernel_triton_b200.rotary_embedding import append_rotary_paged_kv_cache, apply_rotary_qk, rotary_cos_sin, rotary_into

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda"


def test_serving_example_agrees_with_dense_attention():
    spec = importlib.util.spec_from_file_location("paged_serving", os.path.join(ROOT, "examples", "paged_serving.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    _lib.device_status(0, clear=True)
    worst, used = example.main(verbose=False)
    # fp16 rounds each rotated row, weight and output once (2^-11 relative, values below 4)
    assert worst <= 8e-3
    assert used == -(-176 // 16) + -(-44 // 16)  # 100 + 70 + 1 + 5 and 37 + 1 + 1 + 5 tokens, no page shared
    assert _lib.device_status(0) == 0


def test_offsets_past_32_bits():
    # a pool of 4.8 GB; the sequences live in its last pages
    P, Hkv, D, N = 16, 8, 128, 74_000
    pool = torch.zeros((N, 2, Hkv, P, D), dtype=torch.float16, device=DEV)
    small = torch.zeros((8, 2, Hkv, P, D), dtype=torch.float16, device=DEV)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    far, near = [N - 1, N - 5, 3, N - 2, N - 3], [1, 5, 3, 2, 4]
    at, indptr, last = i32([0, 33, 65]), i32([0, 3, 5]), i32([1, 16])  # two sequences of 33 and 32 tokens, all new
    g = torch.Generator(device=DEV).manual_seed(1)
    q, k, v = (torch.randn((65, H, D), generator=g, device=DEV).half() for H in (32, 8, 8))
    table = rotary_cos_sin(64, D, device=DEV)
    outs = []
    for cache, pages in ((pool, far), (small, near)):
        q2 = append_rotary_paged_kv_cache(cache, q, k, v, at, indptr, i32(pages), last, table)
        outs.append((q2, flash_attention_chunk_paged(q2, at, cache, indptr, i32(pages), last)))
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])
    assert torch.equal(pool[torch.tensor(far, device=DEV)], small[torch.tensor(near, device=DEV)])
    copy_kv_pages(pool, i32([N - 1]), i32([N - 10]))
    assert torch.equal(pool[N - 10], small[1])
    t = fork_paged_kv_cache(pool, indptr, i32(far), last, i32([0, 0]))
    assert t[1].tolist() == far[:3] + far[:2] + [0] and torch.equal(pool[0], small[3])
    new, used = compact_paged_kv_cache(pool, i32(far))
    assert int(used) == 5 and new.tolist() == [4, 0, 3, 2, 1]
    assert torch.equal(pool[new.long()], small[torch.tensor(near, device=DEV)])
    # rows whose offsets in q pass 2^31 elements
    T = 2_200_000
    big = torch.empty((T, 1, 1024), dtype=torch.float16, device=DEV)[:, :, :64]
    big[-1] = q[0, 0, :64]
    pos = torch.zeros(T, dtype=torch.int32, device=DEV)
    pos[-1] = 7
    out = torch.empty_like(big)
    rotary_into(out, None, big, None, rotary_cos_sin(8, 64, device=DEV), pos)
    one = apply_rotary_qk(q[:1, :1, :64], k[:1, :1, :64], rotary_cos_sin(8, 64, device=DEV), i32([7]))[0]
    assert torch.equal(out[-1], one[0])
    assert _lib.device_status(0) == 0

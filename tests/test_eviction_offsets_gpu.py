"""The operators for shared prefixes and eviction over a pool whose offsets pass 32 bits: the same bits as in a small one."""
import pytest
import torch

from attention_kernel_triton_b200 import _lib
from attention_kernel_triton_b200.paged_kv_eviction import (accumulate_attention_weights_paged, evict_paged_kv_cache,
                                                            select_kept_tokens)
from attention_kernel_triton_b200.paged_prefix_attention import flash_attention_shared_prefix_paged_with_lse

pytestmark = pytest.mark.gpu
DEV = "cuda"


def same(a, b):
    return bool(torch.equal(a, b))


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("form", ["contiguous", "tokens first"])  # tensor maps of one run, and of strides
def test_far_pages(form):
    _lib.device_status(0, clear=True)
    P, Hkv, D, N = 16, 8, 128, 74_000  # 4.8 GB
    big = torch.zeros((N, 2, Hkv, P, D), dtype=torch.float16, device=DEV)
    if form == "tokens first":
        big = big.view(N, 2, P, Hkv, D).transpose(2, 3)
    small = torch.zeros((16, 2, Hkv, P, D), dtype=torch.float16, device=DEV)
    far = [N - 1, N - 5, 3, N - 2, N - 1, N - 5, N - 9, N - 4, 70_000, 66_000]
    near = [1, 5, 3, 2, 1, 5, 9, 4, 10, 11]
    gen = torch.Generator(device=DEV).manual_seed(1)
    for a, b in zip(far, near):
        small[b] = torch.randn((2, Hkv, P, D), generator=gen, device=DEV).half()
        big[a] = small[b]
    starts, last = i32([0, 4, 8, 10]), i32([9, 16, 3])
    rows, groups, shared = i32([0, 2, 5, 25]), i32([0, 2, 3]), i32([2, 0])
    q = torch.randn((25, 32, D), generator=gen, device=DEV).half()
    out = {}
    for name, pool, pages in (("far", big, far), ("near", small, near)):
        table = (starts, i32(pages), last)
        o, lse = flash_attention_shared_prefix_paged_with_lse(q, rows, pool, *table, groups, shared)
        w = accumulate_attention_weights_paged(None, q, rows, pool, *table, lse, out=torch.zeros(3, Hkv, 64, device=DEV))
        keep, kept = select_kept_tokens(w, i32([57, 64, 19]), 40, sinks=32)
        table = evict_paged_kv_cache(pool, *table, keep, kept, weights=w)
        ids, at = table[1].tolist(), table[0].tolist()
        out[name] = o, lse, keep, kept, w, table[0], table[2], pool[[x for x in ids if x >= 0]].contiguous()
        assert at == [0, 3, 6, 8]
    for a, b in zip(out["far"], out["near"]):
        assert same(a, b)
    assert _lib.device_status(0) == 0

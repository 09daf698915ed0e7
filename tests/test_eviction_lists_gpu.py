"""Eviction with lists that do not ascend: no page of another holder is written."""
import pytest
import torch

from test_paged_kv_eviction_gpu import DEV, i32, same

from attention_kernel_triton_b200 import _lib
from attention_kernel_triton_b200.paged_kv_eviction import evict_paged_kv_cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 5])  # 16-byte pieces, single values
@pytest.mark.parametrize("n", [8, 16, 1024])
@pytest.mark.parametrize("held", ["forked", "reserved"])
def test_a_list_that_does_not_ascend_writes_no_page_of_others(held, n, D):
    P, H, pages = 8, 2, 256
    gen = torch.Generator().manual_seed(n)
    pool = torch.randn(2 * pages, 2, H, P, D, generator=gen).half()
    first = torch.randperm(2 * pages, generator=gen)[:pages].tolist()
    # the other holder of all its pages: a second sequence, which keeps everything, or the mask
    tables = [first, first] if held == "forked" else [first]
    starts, indices = i32([0, pages, 2 * pages][:len(tables) + 1]), i32(sum(tables, []))
    M = max(n, pages * P)
    keep = torch.arange(M, dtype=torch.int32).repeat(len(tables), H, 1)
    # the last entry of every page is in its place, those before it come from far behind
    slots = torch.arange(n)
    far = slots % P != P - 1
    keep[0, :, :n][:, far] = (slots[far] + 900).int()
    mask = None
    if held == "reserved":
        mask = torch.zeros(2 * pages, dtype=torch.bool, device=DEV)
        mask[first] = True
    dev = pool.to(DEV)
    _lib.device_status(0, clear=True)
    evict_paged_kv_cache(dev, starts, indices, i32([P] * len(tables)), keep.to(DEV), i32([n, M][:len(tables)]),
                         reserved=mask)
    assert _lib.device_status(0, clear=True) == 3
    for page in first:
        assert same(dev[page].cpu(), pool[page])


def test_entries_in_order_before_one_that_is_not():
    # slot 0 takes token 4 and the others follow; the last entry names its own slot, below the one before it, and is skipped
    pool = torch.randn(4, 2, 1, 8, 64).half()
    dev, w = pool.to(DEV), torch.rand(1, 1, 16, device=DEV)
    old = w.clone()
    keep = [4, 5, 6, 7, 8, 9, 10, 7]
    _lib.device_status(0, clear=True)
    got = evict_paged_kv_cache(dev, i32([0, 2]), i32([2, 1]), i32([8]), i32(keep).view(1, 1, 8), i32([8]), weights=w)
    assert _lib.device_status(0, clear=True) == 3
    assert got[1].tolist() == [2]
    rows = torch.cat((pool[2], pool[1]), 2)
    assert same(dev[2, :, :, :7].cpu(), rows[:, :, keep[:7]]) and same(dev[2, :, :, 7].cpu(), pool[2, :, :, 7])
    assert same(w[0, 0, :7], old[0, 0, keep[:7]]) and same(w[0, 0, 7], old[0, 0, 7]) and (w[0, 0, 8:] == 0).all()

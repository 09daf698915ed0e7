"""Eviction with lists that do not ascend."""
import pytest
import torch

from test_paged_kv_eviction_gpu import DEV, i32, same

from attention_kernel_triton_b200 import _lib
from attention_kernel_triton_b200.paged_kv_eviction import evict_paged_kv_cache

pytestmark = pytest.mark.gpu


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

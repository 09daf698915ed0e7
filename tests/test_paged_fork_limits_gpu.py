"""Forks at their limits: more entries than the buffer, and than 32 bits, hold; a last page outside the pool."""
import pytest
import torch

from attention_kernel_triton_b200 import _lib
from attention_kernel_triton_b200.paged_kv_pages import fork_paged_kv_cache

pytestmark = pytest.mark.gpu
DEV = "cuda"


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def test_sums_of_entries_past_32_bits():
    # 1024 children of 2.2M entries each are 2.25e9 entries: cut by max_entries all the same
    _lib.device_status(0, clear=True)
    n, F, most = 2_200_000, 1024, 1000
    pool = torch.zeros((4, 2, 2, 1, 16), dtype=torch.float16, device=DEV)
    indices = (torch.arange(n, device=DEV) % 4).int()
    parents = torch.zeros(F, dtype=torch.int32, device=DEV)
    starts, out, last = fork_paged_kv_cache(pool, i32([0, n]), indices, i32([1]), parents, max_entries=most)
    assert starts.tolist() == [0] + [most] * F
    assert torch.equal(out, indices[:most]) and last.tolist() == [1] + [0] * (F - 1)
    assert _lib.device_status(0, clear=True) == 5


def test_last_pages_outside_the_pool_are_kept_by_every_child():
    _lib.device_status(0, clear=True)
    pool = torch.randn((8, 2, 1, 4, 16), device=DEV).half()
    before = pool.clone()
    for bad in (1 << 20, -7):
        t = fork_paged_kv_cache(pool, i32([0, 2, 4]), i32([3, bad, 5, 6]), i32([2, 4]), i32([0, 0, 1, 0]))
        assert t[1].tolist() == [3, bad, 3, bad, 5, 6, 3, bad] and t[2].tolist() == [2, 2, 4, 2]
        assert torch.equal(pool, before)
        assert _lib.device_status(0, clear=True) == 2

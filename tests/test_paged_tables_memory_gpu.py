"""What the tables that the page operators return keep alive."""
import pytest
import torch

from attention_kernel_triton_b200.paged_kv_pages import compact_paged_kv_cache, fork_paged_kv_cache

pytestmark = pytest.mark.gpu
DEV = "cuda"


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def test_tables_do_not_keep_the_workspace():
    N = 200_000
    pool = torch.zeros((N, 2, 1, 1, 8), dtype=torch.float16, device=DEV)
    live = i32([7, 199_999, 3])
    new, used = compact_paged_kv_cache(pool, live)
    assert new.untyped_storage().nbytes() + used.untyped_storage().nbytes() <= 64
    t = fork_paged_kv_cache(pool, i32([0, 3]), live, i32([1]), i32([0, 0]), max_entries=6)
    assert max(x.untyped_storage().nbytes() for x in t) <= 128

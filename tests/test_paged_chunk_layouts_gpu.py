"""Chunk attention's refusals and copies of layouts: a call that cannot be served does not copy the pool first."""
import pytest
import torch

from attention_kernel_triton_b200 import _lib
from attention_kernel_triton_b200.paged_chunk_attention import chunk_paged_into, flash_attention_chunk_paged

pytestmark = pytest.mark.gpu
DEV, FP16 = "cuda", torch.float16


def test_refused_and_copied_layouts_leave_the_pool_where_it_is():
    def pool_of(D, P=16, N=512):  # token-major pages, 32 MB and more
        return torch.zeros((N, 2, P, 8, D), dtype=FP16, device=DEV).transpose(2, 3)

    def args(D):
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
        return i32([0, 2]), pool_of(D), i32([0, 3]), i32([5, 6, 7]), i32([16])

    def grown(call):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        call()
        return torch.cuda.max_memory_allocated() - before

    def refused(q, rest, out=None):
        def call():
            with pytest.raises(_lib.AktError):
                chunk_paged_into(torch.empty_like(q) if out is None else out, q, *rest)
        return call

    small = 8 << 20
    for D in (96, 256):  # head_dim
        rest = args(D)
        assert grown(refused(torch.zeros((2, 8, D), dtype=FP16, device=DEV), rest)) < small
    rest = args(128)
    q = torch.zeros((2, 8, 128), dtype=FP16, device=DEV)
    odd = torch.zeros((2, 8, 129), dtype=FP16, device=DEV)[:, :, 1:]
    assert grown(refused(q, rest, out=odd)) < small
    assert grown(refused(torch.zeros((2, 8 * 129, 128), dtype=FP16, device=DEV), rest)) < small  # 129 heads per kv head
    # queries off the 16-byte grid are copied, the pool is not
    odd.normal_()
    assert grown(lambda: flash_attention_chunk_paged(odd, *rest)) < small
    assert torch.equal(flash_attention_chunk_paged(odd, *rest), flash_attention_chunk_paged(odd.contiguous(), *rest))
    # a pool off the grid is
    wide = torch.randn((12, 2, 8, 16, 129), device=DEV).half()[..., 1:]
    got = flash_attention_chunk_paged(odd, rest[0], wide, *rest[2:])
    assert torch.equal(got, flash_attention_chunk_paged(odd, rest[0], wide.contiguous(), *rest[2:]))
    # and so are contiguous ones that start off it
    flat = torch.randn(1 + wide.numel(), device=DEV).half()[1:]
    moved, q1 = flat.view(wide.shape), torch.randn(1 + odd.numel(), device=DEV).half()[1:].view(odd.shape)
    got = flash_attention_chunk_paged(q1, rest[0], moved, *rest[2:])
    assert torch.equal(got, flash_attention_chunk_paged(q1.clone(), rest[0], moved.clone(), *rest[2:]))


def test_pools_with_heads_that_are_one():
    # a head's pages given to every head by a stride of zero, beside queries off the grid
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    one = torch.randn((6, 2, 1, 16, 64), device=DEV).half()
    pool, q = one.expand(6, 2, 4, 16, 64), torch.randn((3, 8, 65), device=DEV).half()[..., 1:]
    rest = (i32([0, 2]), i32([4, 1]), i32([9]))
    got = flash_attention_chunk_paged(q, i32([0, 3]), pool, *rest)
    assert torch.equal(got, flash_attention_chunk_paged(q.contiguous(), i32([0, 3]), pool.contiguous(), *rest))

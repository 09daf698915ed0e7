"""Chunk attention where parts of a row meet: weights of exactly zero, other batches around a sequence."""
import math

import pytest
import torch

from attention_kernel_triton_b200 import _lib
from attention_kernel_triton_b200.paged_chunk_attention import (flash_attention_chunk_paged,
                                                                flash_attention_chunk_paged_with_lse)
from test_paged_chunk_gpu import BF16, DEV, FP16, Case

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def device_status_clean():
    _lib.device_status(0, clear=True)
    yield


def set_row(c, pos, kv, value, dim):
    c.pool[int(c.indices[pos // c.P]), kv, :, pos % c.P, dim] = value


@pytest.mark.parametrize("B", [1, 40])
@pytest.mark.parametrize("D", [64, 128])
def test_values_that_are_not_finite_behind_a_weight_of_zero(D, B):
    # the first half of the keys scores 200 below the second, so their weights are 0 in 32 bits; a value there that is
    # not finite still makes the row's not finite, however the sequences are cut over the CTAs
    L = 8192 if B == 1 else 1024
    c = Case([L] * B, [2] * B, Hkv=1, G=4, D=D, seed=1)
    c.q.fill_(1.0)
    far = 100.0 / math.sqrt(D)  # scores of +-100: D far / sqrt(D)
    c.pool[:, 0] = far
    for p in c.indices.view(B, -1)[:, :L // 2 // c.P].flatten().tolist():
        c.pool[p, 0] = -far
    c.pool[:, 1] = 1.0
    clean = flash_attention_chunk_paged(*c.args())
    assert (clean == 1).all()
    set_row(c, 5, 1, math.nan, 3)
    set_row(c, 700 if B == 1 else 70, 1, math.inf, 7)
    got, lse = flash_attention_chunk_paged_with_lse(*c.args())
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[:2, :, [3, 7]] = True
    assert torch.equal(~torch.isfinite(got), bad)
    assert (got[~bad] == 1).all() and torch.isfinite(lse).all()


@pytest.mark.parametrize("dtype,D", [(FP16, 128), (BF16, 64)])
def test_a_sequence_alone_and_among_others(dtype, D):
    lens, news = [700, 300, 90, 2500, 16], [10, 300, 90, 3, 1]
    c = Case(lens, news, Hkv=2, G=4, D=D, dtype=dtype, seed=3)
    at, ind = c.at.tolist(), c.indptr.tolist()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731

    def batch(order):
        O, lse = torch.empty_like(c.q), torch.empty(c.q.shape[:2], device=DEV)
        starts = lambda counts: i32([0, *torch.tensor(counts).cumsum(0).tolist()])  # noqa: E731
        got, l = flash_attention_chunk_paged_with_lse(
            torch.cat([c.q[at[b]:at[b + 1]] for b in order]), starts([news[b] for b in order]), c.pool,
            starts([ind[b + 1] - ind[b] for b in order]), torch.cat([c.indices[ind[b]:ind[b + 1]] for b in order]),
            c.last[order])
        r = 0
        for b in order:
            O[at[b]:at[b + 1]], lse[at[b]:at[b + 1]] = got[r:r + news[b]], l[r:r + news[b]]
            r += news[b]
        return O, lse

    for order in ([0, 1, 2, 3, 4], [4, 2, 0, 3, 1], [1, 4, 3, 0, 2]):
        c.close(*batch(order), True)
    alone = [batch([b]) for b in range(5)]
    rows = [slice(at[b], at[b + 1]) for b in range(5)]
    c.close(torch.cat([alone[b][0][rows[b]] for b in range(5)]), torch.cat([alone[b][1][rows[b]] for b in range(5)]), True)
    assert _lib.device_status(0) == 0

"""Accumulated attention weights where keys, queries or log-sum-exps are at their limits, and what a call copies."""
import math

import pytest
import torch

from test_attention_weights_gpu import DEV, check, make, reference_lse, same

from attention_kernel_triton_b200.paged_kv_eviction import accumulate_attention_weights_paged

pytestmark = pytest.mark.gpu


def key_place(c, b, j):
    """Page and row of key j of sequence b."""
    P = c["cache"].shape[3]
    return int(c["indices"][int(c["starts"][b]) + j // P]), j % P


@pytest.mark.parametrize("dtype,D", [(torch.float16, 64), (torch.bfloat16, 128)])
@pytest.mark.parametrize("G", [1, 3, 5, 6, 7, 12, 28, 33, 64, 65, 96, 100])
def test_a_key_that_every_row_scores_minus_infinity_gets_nothing(G, dtype, D):
    # half tiles full of tokens, whose last columns no row fills where 128 is no multiple of the group
    for n in (128 // G, 2 * (128 // G), 5 * (128 // G)):
        c = make([n + 300], [n], G, 1, D, 16, dtype, seed=G)
        c["q"][..., 3] = c["q"][..., 3].abs() + 0.125
        for j in (0, 7, 200, n + 40):
            page, row = key_place(c, 0, j)
            c["cache"][page, 0, :, row, 3] = -math.inf
        for causal in (True, False):
            start = torch.rand(1, 1, n + 300, device=DEV)
            got = check(c, causal, start=start)
            assert torch.isfinite(got).all()
            for j in (0, 7, 200, n + 40):
                assert got[0, 0, j] == start[0, 0, j]


@pytest.mark.parametrize("Hq,Hkv", [(4, 1), (6, 2), (1, 1)])
def test_a_row_whose_lse_is_minus_infinity_adds_nothing_whatever_it_holds(Hq, Hkv):
    c = make([300, 200], [70, 200], Hq, Hkv, 64, 16, seed=20)
    lse = reference_lse(c, True, 0.125)
    off = torch.zeros(270, dtype=torch.bool, device=DEV)
    off[[0, 1, 33, 69, 70, 71, 140, 269]] = True
    lse[off] = -math.inf
    c["q"][off] = math.nan
    c["q"][1] = math.inf
    got = check(c, lse=lse)
    assert torch.isfinite(got).all()
    # a head of a row alone
    c = make([90], [40], 4, 1, 128, 8, seed=21)
    lse = reference_lse(c, False, 128 ** -0.5)
    lse[5, 2] = -math.inf
    c["q"][5, 2] = math.nan
    assert torch.isfinite(check(c, False, lse=lse)).all()


@pytest.mark.parametrize("n,G", [(1, 1), (1, 4), (5, 1), (40, 2), (130, 1)])
def test_weights_past_the_range_of_fp32_are_infinite(n, G):
    # log-sum-exps that are not the rows' own: 60 below them (weights up to e^60), then 100 (past fp32)
    c = make([300], [n], G, 1, 64, 16, seed=22, scale=0.125)
    lse = reference_lse(c, False, 0.125)
    check(c, False, lse=lse - 60)
    args = c["q"], c["at"], c["cache"], c["starts"], c["indices"], c["last"]
    for far in (100, 1000):
        got = accumulate_attention_weights_paged(None, *args, lse - far, causal=False, out=torch.zeros(1, 1, 300, device=DEV))
        assert (got == math.inf).all()  # exp(-|q k| - log 300 + 100) > e^89
    # a key that every row scores +infinity, beside finite ones
    c["q"][..., 0] = 1
    page, row = key_place(c, 0, 17)
    c["cache"][page, 0, 0, row, 0] = math.inf
    got = accumulate_attention_weights_paged(None, *args, lse, causal=False, out=torch.zeros(1, 1, 300, device=DEV))
    assert got[0, 0, 17] == math.inf and torch.isfinite(got[0, 0, :17]).all() and torch.isfinite(got[0, 0, 18:]).all()


def test_queries_off_the_grid_are_copied_and_the_pool_is_not():
    c = make([300, 90], [40, 1], 8, 8, 128, 16, seed=23)
    args = c["at"], c["starts"], c["indices"], c["last"], reference_lse(c, True, 128 ** -0.5)

    def run(q, pool):
        return accumulate_attention_weights_paged(None, q, args[0], pool, *args[1:], out=torch.zeros(2, 8, 300, device=DEV))

    want = run(c["q"], c["cache"])
    pool = torch.zeros(600, *c["cache"].shape[1:], dtype=c["cache"].dtype, device=DEV)  # 39 MB
    pool[:c["cache"].shape[0]] = c["cache"]
    flat = torch.zeros(c["q"].numel() + 1, dtype=c["q"].dtype, device=DEV)
    shifted = flat[1:].view(c["q"].shape)  # contiguous, and off the grid
    odd = torch.zeros(*c["q"].shape[:2], 129, dtype=c["q"].dtype, device=DEV)[..., 1:]
    for q in (shifted, odd):
        q.copy_(c["q"])
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        got = run(q, pool)
        assert same(got, want)
        assert torch.cuda.max_memory_allocated() - before < 8 << 20
    flat = torch.zeros(c["cache"].numel() + 1, dtype=c["cache"].dtype, device=DEV)
    moved = flat[1:].view(c["cache"].shape)
    moved.copy_(c["cache"])
    assert same(run(shifted, moved), want) and same(run(c["q"], moved), want)

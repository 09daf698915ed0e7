"""Pages of a paged cache against the same bookkeeping in plain Python: copy, fork (copy on write), compact, free."""
import random

import pytest
import torch

from attention_kernel_triton_b200 import _lib
from attention_kernel_triton_b200 import workloads as W
from attention_kernel_triton_b200.decode_flash_attention_redundant_var_len_paged import flash_attention_decode_paged
from attention_kernel_triton_b200.paged_kv_pages import (compact_paged_kv_cache, copy_kv_pages, fork_paged_kv_cache,
                                                         free_kv_pages)

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def device_status_clean():
    _lib.device_status(0, clear=True)
    yield


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def make(lens, P, Hkv=2, D=64, layers=None, extra=0, seed=0, dtype=torch.float16):
    g = torch.Generator().manual_seed(seed)
    n = sum(-(-L // P) for L in lens)
    perm = torch.randperm(n + extra, generator=g)[:n].to(torch.int32)
    indptr, _, last, _, _, _ = W.paged_layout_from_lens(lens, P, g)
    shape = (n + extra, 2, Hkv, P, D) if layers is None else (layers, n + extra, 2, Hkv, P, D)
    pool = torch.randn(shape, generator=g).to(dtype).to(DEV)
    return pool, indptr.to(DEV), perm.to(DEV), last.to(DEV)


def fork_ref(pool, indptr, indices, last, parents, P, reserved=None):
    """(indptr, indices, last, pool) after the fork, by the rules."""
    pool = pool.clone()
    layers = pool if pool.dim() == 6 else pool[None]
    N = layers.shape[1]
    indptr, indices, last = indptr.tolist(), indices.tolist(), last.tolist()
    pages = [indices[indptr[b]:indptr[b + 1]] for b in range(len(last))]
    live = set(p for b in parents for p in pages[b]) | (set(reserved) if reserved else set())
    dead = [p for p in range(N) if p not in live]
    oi, ox, ol, seen = [0], [], [], set()
    for b in parents:
        mine = list(pages[b])
        if b in seen and mine and last[b] < P:
            to = dead.pop(0) if dead else -1
            if to >= 0:
                layers[:, to] = layers[:, mine[-1]]
            mine[-1] = to
        seen.add(b)
        ox += mine
        oi.append(len(ox))
        ol.append(last[b])
    return oi, ox, ol, pool


def same(got, want):
    assert [t.tolist() for t in got[:3]] == [list(x) for x in want[:3]]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("P,Hkv,D,layers", [(16, 8, 128, None), (5, 2, 64, 3), (1, 1, 64, None), (64, 2, 80, 2), (7, 3, 5, None)])
def test_fork_matches_plain(P, Hkv, D, layers, dtype):
    lens = [1, P, 3 * P + 1, 0, 2 * P - 1 if P > 1 else 2, 5 * P, 4]
    pool, indptr, indices, last = make(lens, P, Hkv, D, layers, extra=6, seed=P, dtype=dtype)
    parents = [2, 4, 2, 0, 3, 3, 5, 5, 2, 6]
    want = fork_ref(pool, indptr, indices, last, parents, P)
    got = fork_paged_kv_cache(pool, indptr, indices, last, i32(parents))
    same(got, want)
    assert torch.equal(pool, want[3])
    assert all(t.dtype == torch.int32 for t in got)
    # again on the same table: the same result
    again = fork_paged_kv_cache(pool, indptr, indices, last, i32(parents), max_entries=got[1].numel() + 3)
    assert again[1].tolist() == got[1].tolist() + [-1] * 3 and torch.equal(again[0], got[0])
    assert torch.equal(pool, want[3])
    assert _lib.device_status(0) == 0


def test_fork_of_many_random_batches():
    rng = random.Random(7)
    for k in range(12):
        P = rng.choice((1, 4, 16))
        B, F = rng.choice((1, 3, 40, 1100)), rng.choice((0, 1, 5, 300, 1500))
        lens = [rng.choice((0, 1, P, 2 * P, rng.randrange(1, 6 * P + 1))) for _ in range(B)]
        pool, indptr, indices, last = make(lens, P, 1, 8, extra=F + rng.randrange(50), seed=k)
        N = pool.shape[0]
        parents = [rng.randrange(B) for _ in range(F)]
        named = set(indices.tolist())
        keep = [p for p in range(N) if p not in named and rng.random() < 0.2]
        spare = N - len(named) - len(keep)
        mask = torch.zeros(N, dtype=torch.bool)
        mask[keep] = True
        want = fork_ref(pool, indptr, indices, last, parents, P, keep)
        got = fork_paged_kv_cache(pool, indptr, indices, last, i32(parents), reserved=mask.to(DEV))
        same(got, want)
        assert torch.equal(pool, want[3])
        assert _lib.device_status(0, clear=True) == (6 if -1 in want[1] else 0), spare


def test_fork_decodes_like_its_parents():
    lens = [37, 50, 16]
    c = W.make_paged(B=3, Hq=8, Hkv=2, D=128, page_size=16, lens=lens, seed=3, device=DEV, extra_pages=4)
    parents = i32([1, 0, 1, 0, 2, 1])
    t = fork_paged_kv_cache(c.cache, c.indptr, c.indices, c.last_page_len, parents)
    q = c.q[parents.long()]
    O = flash_attention_decode_paged(q, c.cache, *t)
    ref = flash_attention_decode_paged(c.q, c.cache, c.indptr, c.indices, c.last_page_len)[parents.long()]
    assert torch.equal(O, ref)


def test_fork_cut_and_bad_tables():
    P = 16
    pool, indptr, indices, last = make([20, 40, 64], P, extra=4, seed=1)
    before = pool.clone()
    want = fork_ref(pool, indptr, indices, last, [1, 0, 1], P)
    # room for five entries of eight: the children past them are cut, and a cut child needs no page
    got = fork_paged_kv_cache(pool, indptr, indices, last, i32([1, 0, 1]), max_entries=6)
    assert got[0].tolist() == [0, 3, 5, 6] and got[2].tolist() == [8, 4, P]
    assert got[1].tolist() == want[1][:5] + [indices.tolist()[2]]
    assert torch.equal(pool, before)
    assert _lib.device_status(0, clear=True) == 5
    # parents outside the batch
    got = fork_paged_kv_cache(pool, indptr, indices, last, i32([0, 3, -1, 2]), max_entries=6)
    assert got[0].tolist() == [0, 2, 2, 2, 6] and got[2].tolist() == [4, 0, 0, 16]
    assert _lib.device_status(0, clear=True) == 4
    # a page id outside the pool is kept and recorded, and nothing is copied from it
    bad = indices.clone()
    bad[1] = 1 << 20
    got = fork_paged_kv_cache(pool, indptr, bad, last, i32([0, 0]), max_entries=4)
    assert got[1].tolist()[:3] == [int(indices[0]), 1 << 20, int(indices[0])]
    assert torch.equal(pool, before)
    assert _lib.device_status(0, clear=True) == 2
    # bounds past the index array
    got = fork_paged_kv_cache(pool, i32([0, 2, 5, 99]), indices, last, i32([2, 0]), max_entries=2)
    assert got[0].tolist() == [0, 0, 2]
    assert _lib.device_status(0, clear=True) == 4
    # no dead page left
    pool, indptr, indices, last = make([20, 17], P, extra=1, seed=2)
    got = fork_paged_kv_cache(pool, indptr, indices, last, i32([0, 1, 0, 1]))
    assert got[1].tolist().count(-1) == 1 and got[1].tolist()[-1] == -1
    assert _lib.device_status(0, clear=True) == 6


def compact_ref(pool, indices, reserved=()):
    pool = pool.clone()
    layers = pool if pool.dim() == 6 else pool[None]
    N = layers.shape[1]
    res = set(reserved)
    live = sorted(set(p for p in indices.tolist() if 0 <= p < N and p not in res))
    targets = [p for p in range(N) if p not in res][:len(live)]
    holes = [p for p in targets if p not in set(live)]
    movers = [p for p in live if p not in set(targets)]
    old = layers.clone()
    to = dict(zip(movers, holes))
    for s, d in to.items():
        layers[:, d] = old[:, s]
    used = max([p + 1 for p in targets] + [p + 1 for p in res] + [0])
    return [to.get(p, p) for p in indices.tolist()], used, pool


@pytest.mark.parametrize("P,Hkv,D,layers", [(16, 8, 128, None), (5, 2, 64, 3), (1, 1, 64, None), (7, 3, 5, 2)])
def test_compact_matches_plain(P, Hkv, D, layers):
    lens = [3 * P + 1, 2, 5 * P, P, 40]
    pool, indptr, indices, last = make(lens, P, Hkv, D, layers, extra=9, seed=P)
    at = indptr.tolist()
    stay = torch.cat([indices[at[b]:at[b + 1]] for b in (0, 2, 4)])
    shared = torch.cat((stay, stay[:3], i32([-1])))  # shared pages appear twice, a -1 stays
    want = compact_ref(pool, shared)
    new, used = compact_paged_kv_cache(pool, shared)
    assert new.tolist() == want[0] and int(used) == want[1] and used.shape == ()
    assert torch.equal(pool, want[2])
    assert int(used) == len(set(stay.tolist())) == int(new.max()) + 1
    again, _ = compact_paged_kv_cache(pool, shared)
    assert torch.equal(again, new) and torch.equal(pool, want[2])
    still, used2 = compact_paged_kv_cache(pool, new)
    assert torch.equal(still, new) and int(used2) == int(used)
    assert _lib.device_status(0) == 0


def test_compact_random_pools_with_reserved_pages():
    rng = random.Random(11)
    for k in range(12):
        N = rng.choice((1, 31, 32, 33, 1000, 40000))
        pool = torch.randn(N, 2, 1, 1, 8, device=DEV).half()
        share = rng.choice((0.0, 0.05, 0.5, 0.95, 1.0))
        live = [p for p in range(N) if rng.random() < share]
        rng.shuffle(live)
        res = [p for p in range(N) if rng.random() < rng.choice((0.0, 0.1, 0.6))]
        mask = torch.zeros(N, dtype=torch.bool)
        mask[res] = True
        idx = i32(live)
        want = compact_ref(pool, idx, res)
        new, used = compact_paged_kv_cache(pool, idx, reserved=mask.to(DEV))
        assert new.tolist() == want[0] and int(used) == want[1]
        assert torch.equal(pool, want[2])
        pages, count = free_kv_pages(N, idx, reserved=mask.to(DEV))
        dead = sorted(set(range(N)) - set(live) - set(res))
        assert int(count) == len(dead) and pages.tolist() == dead + [-1] * (N - len(dead))
    assert _lib.device_status(0) == 0


def test_pools_past_the_shared_bitmap():
    # more pages than the plan's bitmaps in shared memory hold
    N = 800_000
    pool = torch.arange(N, device=DEV).to(torch.float16)[:, None, None, None, None].expand(N, 2, 1, 1, 4).contiguous()
    before = pool.clone()
    live = i32([N - 1, 5, 0, N - 7, 3, 123_456])
    new, used = compact_paged_kv_cache(pool, live)
    want, n, _ = compact_ref(torch.zeros(N, 2, 1, 1, 1), live)
    assert new.tolist() == want and int(used) == n == 6
    assert torch.equal(pool[new.long()], before[live.long()])
    pages, count = free_kv_pages(N, live)
    assert int(count) == N - 6 and pages[:5].tolist() == [1, 2, 4, 6, 7] and int(pages[-7]) == N - 2
    t = fork_paged_kv_cache(before, i32([0, 6]), live, i32([0]), i32([0, 0]), max_entries=12)
    assert t[1].tolist() == live.tolist() + live.tolist()[:5] + [1]
    assert torch.equal(before[1], before[123_456])
    assert _lib.device_status(0) == 0


def test_compact_records_bad_ids_and_keeps_them():
    pool = torch.randn(8, 2, 1, 4, 16, device=DEV).half()
    new, used = compact_paged_kv_cache(pool, i32([7, 99, 2]))
    assert new.tolist() == [0, 99, 1] or new.tolist() == [1, 99, 0]
    assert int(used) == 2
    assert _lib.device_status(0) == 2


@pytest.mark.parametrize("layout", ["heads_last", "slice", "odd_start"])
def test_strided_pools(layout):
    P, Hkv, D = 4, 2, 16
    pool, indptr, indices, last = make([9, 6], P, Hkv, D, extra=3, seed=5)
    if layout == "heads_last":  # token-major pages
        mine = pool.transpose(2, 3).contiguous().transpose(2, 3)
    elif layout == "slice":  # a part of a wider head
        wide = torch.zeros(*pool.shape[:-1], 24, dtype=pool.dtype, device=DEV)
        mine = wide[..., 8:]
        mine.copy_(pool)
    else:  # rows that start off the 16-byte grid
        wide = torch.zeros(*pool.shape[:-1], 19, dtype=pool.dtype, device=DEV)
        mine = wide[..., 3:]
        mine.copy_(pool)
    assert not mine.is_contiguous()
    par = [1, 1, 0, 0]
    want = fork_ref(pool, indptr, indices, last, par, P)
    same(fork_paged_kv_cache(mine, indptr, indices, last, i32(par)), want)
    assert torch.equal(mine, want[3])
    copy_kv_pages(mine, i32([0, 1]), i32([2, 3]))
    assert torch.equal(mine[2:4], want[3][0:2])
    want = compact_ref(mine, indices[:2])
    new, used = compact_paged_kv_cache(mine, indices[:2])
    assert new.tolist() == want[0] and torch.equal(mine, want[2])


def test_copy_pages_skips_bad_ids():
    pool = torch.randn(2, 6, 2, 1, 4, 16, device=DEV).bfloat16()
    before = pool.clone()
    copy_kv_pages(pool, i32([0, 6, 1, -1]), i32([4, 2, 77, 3]))
    before[:, 4] = before[:, 0]
    assert torch.equal(pool, before)
    assert _lib.device_status(0) == 2
    copy_kv_pages(pool, i32([]), i32([]))
    assert torch.equal(pool, before)


def test_pages_on_another_stream_and_in_a_graph():
    pool, indptr, indices, last = make([20, 33], 16, extra=4, seed=6)
    par = i32([0, 0, 1, 1])
    want = fork_ref(pool, indptr, indices, last, par.tolist(), 16)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = fork_paged_kv_cache(pool, indptr, indices, last, par, max_entries=10)
    s.synchronize()
    same(got, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = fork_paged_kv_cache(pool, indptr, indices, last, par, max_entries=10)
        new, used = compact_paged_kv_cache(pool, got[1])
    g.replay()
    torch.cuda.synchronize()
    same(got, want)
    assert sorted(set(new.tolist())) == list(range(int(used)))

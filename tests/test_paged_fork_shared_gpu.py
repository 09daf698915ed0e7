"""Forks of pages that several hold: a partly filled last page that `reserved` or another sequence keeps is copied, also
for a parent's first child."""
import random

import pytest
import torch

from attention_kernel_triton_b200 import _lib
from attention_kernel_triton_b200.paged_kv_append import append_paged_kv_cache
from attention_kernel_triton_b200.paged_kv_pages import fork_paged_kv_cache

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def device_status_clean():
    _lib.device_status(0, clear=True)
    yield


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def table_of(seqs, P):
    """The table of sequences given as (pages, tokens)."""
    at = [0]
    for pages, _ in seqs:
        at.append(at[-1] + len(pages))
    last = [n - P * (len(pages) - 1) if pages else 0 for pages, n in seqs]
    return i32(at), i32([p for pages, _ in seqs for p in pages]), i32(last)


def fork_ref(pool, seqs, parents, P, reserved=()):
    """(pages of each child, pool): a partly filled last page stays with the first child that has it as its own last page,
    and with nobody when it is reserved or holds a whole page of a named parent."""
    pool = pool.clone()
    held, partial = set(reserved), set()
    for b in set(parents):
        pages, n = seqs[b]
        full = n // P
        held |= set(pages[:full])
        partial |= set(pages[full:])
    dead = [p for p in range(pool.shape[0]) if p not in held | partial]
    out, keeper, short = [], {}, 0
    for c, b in enumerate(parents):
        pages, n = list(seqs[b][0]), seqs[b][1]
        if pages and n % P:
            x = pages[-1]
            if x in held or keeper.setdefault(x, c) != c:
                pages[-1] = dead.pop(0) if dead else -1
                if pages[-1] >= 0:
                    pool[pages[-1]] = pool[x]
                else:
                    short += 1
        out.append(pages)
    return out, pool, short


def check(pool, seqs, parents, P, reserved=()):
    want, want_pool, short = fork_ref(pool, seqs, parents, P, reserved)
    mask = None
    if reserved:
        mask = torch.zeros(pool.shape[0], dtype=torch.bool, device=DEV)
        mask[list(reserved)] = True
    starts, indices, last = fork_paged_kv_cache(pool, *table_of(seqs, P), i32(parents), reserved=mask,
                                                max_entries=sum(map(len, want)))
    starts, indices = starts.tolist(), indices.tolist()
    assert [indices[starts[c]:starts[c + 1]] for c in range(len(parents))] == want
    assert last.tolist() == table_of(seqs, P)[2][i32(parents).long()].tolist()
    assert torch.equal(pool, want_pool)
    assert _lib.device_status(0, clear=True) == (6 if short else 0)
    return want


def new_pool(N, P, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn((N, 2, 2, P, 16), generator=g).half().to(DEV)


def test_reserved_prefix_is_forked_twice():
    # a prefix that a store keeps (reserved): two continuations, forked at different times, write their own first rows
    P, prefix = 16, ([3, 5], 20)
    pool = new_pool(12, P)
    before = pool.clone()
    held = torch.zeros(12, dtype=torch.bool, device=DEV)
    held[[3, 5]] = True

    def continued(value):
        table = fork_paged_kv_cache(pool, *table_of([prefix], P), i32([0]), reserved=held)
        rows = torch.full((2, 2, 16), value, dtype=torch.float16, device=DEV)
        last = table[2] + 2  # two tokens more, in the same page
        append_paged_kv_cache(pool, rows, rows, i32([0, 2]), table[0], table[1], last)
        held[table[1].long()] = True
        return table[1].tolist(), last

    a, _ = continued(1.0)
    b, _ = continued(2.0)
    assert a[0] == b[0] == 3 and len({a[1], b[1], 5}) == 3
    assert torch.equal(pool[[3, 5]], before[[3, 5]])
    for pages, value in ((a, 1.0), (b, 2.0)):
        assert torch.equal(pool[pages[1], :, :, :4], before[5, :, :, :4])
        assert (pool[pages[1], :, :, 4:6] == value).all()
    assert _lib.device_status(0) == 0


def test_siblings_cut_back_into_a_shared_page():
    P = 8
    # the first was cut back into a page that is a whole one of the second
    assert check(new_pool(9, P), [([0, 4], 11), ([0, 4, 2], 20)], [0, 1], P) == [[0, 1], [0, 4, 2]]
    # both were cut back into the same page: the first child that has it keeps it
    assert check(new_pool(9, P), [([0, 4], 11), ([0, 4], 14)], [1, 0, 1], P) == [[0, 4], [0, 1], [0, 2]]
    # a holder that no child names does not count
    assert check(new_pool(9, P), [([0, 4], 11), ([0, 4], 14)], [0], P) == [[0, 4]]
    # reserved pages that are whole are shared, not copied
    assert check(new_pool(9, P), [([0, 4], 16), ([0, 5], 9)], [0, 0, 1], P, reserved=(0, 4)) == [[0, 4], [0, 4], [0, 5]]
    # no dead page left for the first child
    assert check(new_pool(3, P), [([0, 1], 9)], [0], P, reserved=(1, 2)) == [[0, -1]]


def test_random_batches_that_share_pages():
    rng = random.Random(3)
    for k in range(30):
        P, N = rng.choice((1, 2, 5, 16)), rng.choice((40, 70, 600))
        free = list(range(N))
        rng.shuffle(free)
        seqs = []
        for _ in range(rng.choice((1, 4, 30, 300))):
            if seqs and rng.random() < 0.6:  # a sibling, cut back or not, that may have pages of its own after it
                pages, n = rng.choice(seqs)
                n = rng.randint(0, n)
                pages = pages[:-(-n // P)]
                if n % P == 0 and free and rng.random() < 0.5:
                    pages, n = pages + [free.pop()], n + rng.randint(1, P)
            else:
                m = min(len(free), rng.randint(0, 4))
                pages = [free.pop() for _ in range(m)]
                n = P * (m - 1) + rng.randint(1, P) if m else 0
            seqs.append((list(pages), n))
        parents = [rng.randrange(len(seqs)) for _ in range(rng.choice((1, 7, 90, 1300)))]
        reserved = tuple(p for p in range(N) if rng.random() < rng.choice((0.0, 0.05, 0.3)))
        check(new_pool(N, P, k), seqs, parents, P, reserved)


def test_shared_pages_past_the_shared_memory_bitmap():
    N, P = 800_000, 4
    pool = torch.arange(N, device=DEV).to(torch.float16)[:, None, None, None, None].expand(N, 2, 1, P, 4).contiguous()
    check(pool, [([700_000, 9], 6), ([700_000, 9], 7), ([5, 700_000], 5)], [0, 1, 2, 0], P, reserved=(0, 1))

"""Choice of kept tokens and eviction from a paged cache against plain bookkeeping, value for value."""
import pytest
import torch

from attention_kernel_triton_b200 import _lib
from attention_kernel_triton_b200.paged_kv_eviction import evict_paged_kv_cache, select_kept_tokens

pytestmark = pytest.mark.gpu
DEV = "cuda"


def same(a, b):
    return bool(torch.equal(a, b))


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.fixture(autouse=True)
def status():
    _lib.device_status(0, clear=True)
    yield
    torch.cuda.synchronize()


# ---------------------------------------------------------------------------
# choice
# ---------------------------------------------------------------------------

def plain_choice(row, n, budget, sinks, recent):
    """Kept tokens of one head (a list of floats), by sorting."""
    if n <= budget:
        return list(range(n))
    forced = list(range(sinks)) + list(range(n - recent, n))
    rest = range(sinks, n - recent)
    heavy = sorted(rest, key=lambda j: (row[j] == row[j], row[j] if row[j] == row[j] else 0.0, -j), reverse=True)
    return sorted(forced + heavy[:budget - sinks - recent])


@pytest.mark.parametrize("B,H,L,budget,sinks,recent", [
    (1, 1, 1, 1, 0, 0), (2, 3, 33, 7, 1, 2), (3, 2, 1000, 999, 0, 0), (1, 8, 5000, 64, 4, 60), (2, 2, 4097, 1024, 64, 100),
    (1, 2, 40000, 33, 0, 0), (1, 1, 70001, 20000, 4, 1000), (40, 4, 700, 100, 0, 99), (1, 3, 50, 0, 0, 0),
    (1, 1, 500000, 1000, 3, 5),
])
def test_choice(B, H, L, budget, sinks, recent):
    gen = torch.Generator().manual_seed(L)
    w = torch.randn(B, H, L, generator=gen)
    w[:, 0] = (w[:, 0] * 2).round() / 4  # many ties, both zeros
    lens = [L] + [int(x) for x in torch.randint(0, L + 1, (B - 1,), generator=gen)]
    ind, kept = select_kept_tokens(w.to(DEV), i32(lens), budget, sinks, recent)
    assert ind.shape == (B, H, budget) and ind.dtype == kept.dtype == torch.int32
    assert kept.tolist() == [min(n, budget) for n in lens]
    for b in range(B):
        for h in range(H):
            want = plain_choice(w[b, h].tolist(), lens[b], budget, sinks, recent)
            assert ind[b, h].tolist() == want + [0] * (budget - len(want)), (b, h)
    assert _lib.device_status(0) == 0


def test_choice_of_odd_values_layers_and_strides():
    inf, nan = float("inf"), float("nan")
    w = torch.full((2, 3, 2, 64), -7.0)
    w[0, 0, 0, :8] = torch.tensor([nan, inf, -inf, 0.0, -0.0, 1e-45, -1e-45, nan])
    w[1, 2, 1, 10:14] = torch.tensor([3e38, -3e38, inf, nan])
    w[1, 0] = nan
    big = torch.zeros(2, 3, 4, 80)
    big[:, :, ::2, 5:69] = w
    view = big.to(DEV)[:, :, ::2, 5:69]
    for budget in (1, 3, 6, 63):
        ind, kept = select_kept_tokens(view, i32([64, 20, 64]), budget)
        for l in range(2):
            for b, n in enumerate((64, 20, 64)):
                for h in range(2):
                    want = plain_choice(w[l, b, h].tolist(), n, budget, 0, 0)
                    assert ind[l, b, h].tolist() == want + [0] * (budget - len(want)), (budget, l, b, h)
    other = w.transpose(2, 3).contiguous().transpose(2, 3).to(DEV)  # no unit stride
    assert same(select_kept_tokens(other, i32([64, 20, 64]), 6)[0], select_kept_tokens(view, i32([64, 20, 64]), 6)[0])


def test_choice_cuts_lengths_outside_the_weights():
    w = torch.rand(2, 1, 10, device=DEV)
    ind, kept = select_kept_tokens(w, i32([12, -3]), 4)
    assert kept.tolist() == [4, 0] and ind[1].tolist() == [[0, 0, 0, 0]]
    assert ind[0, 0].tolist() == plain_choice(w[0, 0].tolist(), 10, 4, 0, 0)
    assert _lib.device_status(0, clear=True) == 3


# ---------------------------------------------------------------------------
# eviction
# ---------------------------------------------------------------------------

def plain_evict(pool, starts, indices, last, keep, kept, P, weights=None, reserved=()):
    """The same on lists and CPU tensors; pool [layers, N, 2, H, P, D]."""
    layers, N, H = pool.shape[0], pool.shape[1], pool.shape[3]
    old, named = pool.clone(), [x for x in indices if x >= 0]
    dead = [x for x in range(N) if x not in set(named) | set(reserved)]
    out_starts, out, out_last = [0], [], []
    for b, n in enumerate(kept):
        mine = indices[starts[b]:starts[b + 1]]
        length = (len(mine) - 1) * P + last[b] if mine else 0
        pages = []
        for e in range(-(-n // P)):
            rows = range(e * P, min((e + 1) * P, n))
            stays = all(keep[l, b, h, i] == i for l in range(layers) for h in range(H) for i in rows)
            shared = named.count(mine[e]) > 1 or mine[e] in reserved
            pages.append(dead.pop(0) if shared and not (stays and len(rows) == P) else mine[e])
        for l in range(layers):
            for h in range(H):
                k = keep[l, b, h, :n].long()
                to = torch.tensor([pages[i // P] for i in range(n)], dtype=torch.long)
                at = torch.tensor([mine[j // P] for j in k.tolist()], dtype=torch.long)
                i = torch.arange(n)
                pool[l, to, :, h, i % P] = old[l, at, :, h, k % P]
                if weights is not None:
                    row = weights[l, b, h]
                    moved = row[k].clone()
                    row[:length] = 0
                    row[:n] = moved
        out += pages
        out_starts.append(len(out))
        out_last.append(n - (len(pages) - 1) * P if pages else 0)
    return out_starts, out, out_last


def case(lens, budget, P, H=2, D=64, layers=1, share=1, dtype=torch.float16, seed=0, spare=0, stay=0):
    """Pool, table, lists and weights; every `share` sequences have the first half of the shortest's pages in common,
    the first `stay` tokens of every list stay."""
    gen = torch.Generator().manual_seed(seed)
    B, starts, indices, last, N = len(lens), [0], [], [], 0
    common = []
    for b, n in enumerate(lens):
        if b % share == 0:
            c = min(lens[b:b + share]) // 2 // P if share > 1 else 0
            common = list(range(N, N + c))
            N += c
        pages = -(-n // P)
        own = pages - len(common)
        indices += common + list(range(N, N + own))
        N += own
        starts.append(len(indices))
        last.append(n - P * (pages - 1) if pages else 0)
    N += spare
    place = torch.randperm(N, generator=gen).tolist()
    indices = [place[x] for x in indices]
    pool = torch.randn(layers, N, 2, H, P, D, generator=gen).to(dtype)
    L = max(max(lens), 1)
    weights = torch.rand(layers, B, H, L, generator=gen)
    keep = torch.zeros(layers, B, H, budget, dtype=torch.int32)
    kept = [min(n, budget) for n in lens]
    for l in range(layers):
        for b, n in enumerate(lens):
            for h in range(H):
                s = min(stay, kept[b])
                rest = (torch.randperm(n - s, generator=gen)[:kept[b] - s] + s).sort().values
                keep[l, b, h, :kept[b]] = torch.cat((torch.arange(s), rest))
    return pool, starts, indices, last, keep, kept, weights


def check(c, P, reserved=None, layered=None, pool_dev=None, weights=True):
    pool, starts, indices, last, keep, kept, w = c
    layered = pool.shape[0] > 1 if layered is None else layered
    cut = (lambda t: t) if layered else (lambda t: t[0])
    dev_pool = cut(pool).to(DEV) if pool_dev is None else pool_dev
    dev_w = cut(w).to(DEV) if weights else None
    mask = None
    if reserved is not None:
        mask = torch.zeros(pool.shape[1], dtype=torch.bool, device=DEV)
        mask[list(reserved)] = True
    got = evict_paged_kv_cache(dev_pool, i32(starts), i32(indices), i32(last), cut(keep).to(DEV), i32(kept), weights=dev_w,
                               reserved=mask)
    a, b, c = plain_evict(pool, starts, indices, last, keep, kept, P, w, reserved or ())
    assert got[0].tolist() == a and got[2].tolist() == c
    assert got[1][:len(b)].tolist() == b and set(got[1][len(b):].tolist()) <= {-1}
    assert same(dev_pool.cpu(), cut(pool))
    if weights:
        assert same(dev_w.cpu(), cut(w))
    assert _lib.device_status(0) == 0


@pytest.mark.parametrize("lens,budget,P,kw", [
    ([1], 1, 1, {}),
    ([5, 0, 17], 4, 4, dict(dtype=torch.bfloat16)),
    ([100, 37, 5, 64], 33, 16, dict(H=3)),
    ([300, 41], 64, 20, dict(layers=3, D=128)),
    ([1000, 999, 5000], 900, 16, dict(D=128)),
    ([20000], 9000, 16, dict(H=1)),          # many chunks of a cluster
    ([4000] * 40, 700, 128, dict(H=2)),      # many heads: a CTA each
    ([700, 700], 699, 5, dict(D=40)),
    ([64, 64, 64, 64], 0, 8, {}),
    ([50, 60], 200, 8, {}),                  # nothing goes
])
def test_evict(lens, budget, P, kw):
    check(case(lens, budget, P, **kw), P)


@pytest.mark.parametrize("stay", [0, 7, 16, 40])
@pytest.mark.parametrize("share", [2, 3])
def test_shared_pages_are_copied_only_where_rows_move(share, stay):
    c = case([200, 150, 90, 200, 171, 64], 70, 8, share=share, stay=stay, spare=60, layers=2)
    check(c, 8)


def test_reserved_pages_are_not_written():
    c = case([100, 40], 30, 8, spare=12)
    named = c[2]
    check(c, 8, reserved=[named[0], named[2], named[15]])


def test_sequence_that_names_a_page_twice():
    c = list(case([64], 20, 8, spare=4))
    c[2][5] = c[2][1]
    check(tuple(c), 8)


def test_table_of_many_pages():  # several planning CTAs
    c = case([9000, 7000, 5000], 3000, 1, H=1, D=64, share=3, spare=9000, stay=100)
    check(c, 1)


@pytest.mark.parametrize("form", ["rows", "heads", "odd"])
def test_strided_pools(form):
    c = case([70, 33], 25, 8, D=64)
    pool = c[0][0]
    N, _, H, P, D = pool.shape
    if form == "rows":      # rows of a wider array
        dev = torch.zeros(N, 2, H, P, 80, dtype=pool.dtype, device=DEV)[..., 8:72]
    elif form == "heads":   # tokens before heads
        dev = torch.zeros(N, 2, P, H, D, dtype=pool.dtype, device=DEV).transpose(2, 3)
    else:                   # off the 16-byte grid
        dev = torch.zeros(N, 2, H, P, 67, dtype=pool.dtype, device=DEV)[..., 3:67]
    dev.copy_(pool)
    check(c, 8, pool_dev=dev)


def test_lists_and_weights_of_other_layouts():
    c = case([70, 33], 24, 8, D=64)
    pool, starts, indices, last, keep, kept, w = c
    dev = pool[0].to(DEV)
    wide = torch.zeros(2, 5, 100, device=DEV)
    wide[:, 1:3, 10:80] = w[0].to(DEV)
    long = torch.zeros(2, 2, 40, dtype=torch.int64, device=DEV)
    long[..., :24] = keep[0].to(DEV)
    got = evict_paged_kv_cache(dev, i32(starts).long(), i32(indices).long(), i32(last), long[..., :24], i32(kept),
                               weights=wide[:, 1:3, 10:80])
    plain_evict(pool, starts, indices, last, keep, kept, 8, w)
    assert same(dev.cpu(), pool[0]) and same(wide[:, 1:3, 10:80].cpu(), w[0]) and got[0].dtype == torch.int32
    assert wide[:, 0].abs().sum() == 0 and wide[:, 1:3, :10].abs().sum() == 0 and wide[:, 1:3, 80:].abs().sum() == 0


def test_no_dead_page_left():
    pool, starts, indices, last, keep, kept, w = case([40, 40], 20, 8, share=2, spare=1)
    dev = pool[0].to(DEV)
    got = evict_paged_kv_cache(dev, i32(starts), i32(indices), i32(last), keep[0].to(DEV), i32(kept))
    assert _lib.device_status(0, clear=True) == 6
    pages, dead = got[1].tolist(), (set(range(pool.shape[1])) - set(indices)).pop()
    assert pages.count(dead) == 1 and -1 in pages
    before = pool[0]
    for page in set(indices[:2]):  # shared pages keep their contents
        assert same(dev[page].cpu(), before[page])


def test_bad_lists_and_tables_are_skipped_and_recorded():
    pool, starts, indices, last, keep, kept, w = case([40, 40], 20, 8)
    want = pool.clone()
    good = [(starts, indices, last, keep, kept)]
    for what, status in (("token", 3), ("order", 3), ("count", 3), ("bounds", 4), ("page", 2)):
        k, n, s, ids = keep.clone(), list(kept), list(starts), list(indices)
        if what == "token":
            k[0, 1, 1, 19] = 40
        if what == "order":
            k[0, 1, 0, 5] = k[0, 1, 0, 4]
        if what == "count":
            n[1] = 21
        if what == "bounds":
            s[2] = 99
        if what == "page":
            ids[9] = pool.shape[1] + 5
        dev = pool[0].to(DEV)
        evict_paged_kv_cache(dev, i32(s), i32(ids), i32(last), k[0].to(DEV), i32(n))
        assert _lib.device_status(0, clear=True) == status, what
        # the other sequence is as it would be
        want = pool.clone()
        plain_evict(want, starts, indices, last, keep, kept, 8)
        for page in indices[:starts[1]]:
            assert same(dev[page].cpu(), want[0, page]), what


def test_negative_page_ids_take_no_dead_page():
    # an id below -1 in a sequence beside pages that have to be replaced
    pool, starts, indices, last, keep, kept, w = case([40, 40, 40], 20, 8, share=2, spare=6)
    bad = list(indices)
    bad[starts[2]] = -2
    bad[starts[2] + 1] = -3
    want = pool.clone()
    a, b, c = plain_evict(want, starts[:3], indices[:starts[2]], last[:2], keep[:, :2], kept[:2], 8,
                          reserved=set(bad[starts[2] + 2:]))
    dev = pool[0].to(DEV)
    got = evict_paged_kv_cache(dev, i32(starts), i32(bad), i32(last), keep[0].to(DEV), i32(kept))
    # (the two pages that the bad ids hide are dead: the lowest dead ones are found again)
    dead = sorted(set(range(pool.shape[1])) - {x for x in bad if x >= 0})
    fresh = [x for x in got[1].tolist()[:a[-1]] if x not in indices[:starts[2]]]
    assert fresh == dead[:len(fresh)] and len(fresh) == len(set(fresh)) > 0
    assert got[1].tolist()[a[2]:a[2] + 2] == [-1, -1]
    for b in range(2):  # every row of the good sequences
        pages = got[1].tolist()[a[b]:a[b + 1]]
        mine = indices[starts[b]:starts[b + 1]]
        for h in range(2):
            for i in range(20):
                j = int(keep[0, b, h, i])
                assert same(dev[pages[i // 8], :, h, i % 8].cpu(), pool[0, mine[j // 8], :, h, j % 8])


def test_weights_narrower_than_the_sequences():
    pool, starts, indices, last, keep, kept, w = case([60], 30, 8)
    narrow = w[0, :, :, :40].contiguous()
    dw = narrow.to(DEV)
    evict_paged_kv_cache(pool[0].to(DEV), i32(starts), i32(indices), i32(last), keep[0].to(DEV), i32(kept), weights=dw)
    for h in range(2):
        want = [narrow[0, h, j].item() if j < 40 else 0.0 for j in keep[0, 0, h].tolist()] + [0.0] * 10
        assert dw[0, h].tolist() == want


def test_empty_calls():
    pool = torch.zeros(3, 2, 1, 4, 64, dtype=torch.float16, device=DEV)
    got = evict_paged_kv_cache(pool, i32([0]), i32([]), i32([]), i32([]).view(0, 1, 0), i32([]))
    assert got[0].tolist() == [0] and got[1].numel() == got[2].numel() == 0
    got = evict_paged_kv_cache(pool, i32([0, 0]), i32([2]), i32([0]), i32([[[0]]]), i32([0]))
    assert got[0].tolist() == [0, 0] and got[1].tolist() == [-1] and got[2].tolist() == [0]
    ind, kept = select_kept_tokens(torch.zeros(0, 2, 5, device=DEV), i32([]), 3)
    assert ind.shape == (0, 2, 3) and kept.numel() == 0


def test_graph_and_streams():
    c = case([500, 300], 100, 16, share=2, spare=40)
    pool, starts, indices, last, keep, kept, w = c
    src, dev, dw = pool[0].to(DEV), pool[0].to(DEV), w[0].to(DEV)
    table, lists = (i32(starts), i32(indices), i32(last)), (keep[0].to(DEV), i32(kept))
    lens = i32([500, 300])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            select_kept_tokens(dw, lens, 100)
            evict_paged_kv_cache(dev, *table, *lists, weights=dw)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        chosen = select_kept_tokens(dw, lens, 100)
        got = evict_paged_kv_cache(dev, *table, *lists, weights=dw)
    want_w = w.clone()
    a, b, l = plain_evict(pool, starts, indices, last, keep, kept, 16, want_w)
    for _ in range(2):
        dev.copy_(src)
        dw.copy_(w[0])
        graph.replay()
        torch.cuda.synchronize()
        assert same(dev.cpu(), pool[0]) and same(dw.cpu(), want_w[0])
        assert got[0].tolist() == a and got[1][:len(b)].tolist() == b and got[2].tolist() == l
        assert chosen[0][0, 0].tolist() == plain_choice(w[0, 0, 0].tolist(), 500, 100, 0, 0)

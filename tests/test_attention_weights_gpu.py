"""Accumulated attention weights over a paged cache against the definition in 64 bits."""
import math

import pytest
import torch

from attention_kernel_triton_b200 import _lib
from attention_kernel_triton_b200.paged_chunk_attention import flash_attention_chunk_paged_with_lse
from attention_kernel_triton_b200.paged_kv_eviction import accumulate_attention_weights_paged

pytestmark = pytest.mark.gpu
DEV = "cuda"


def same(a, b):
    return bool(torch.equal(a, b))


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def make(lens, news, Hq, Hkv, D, P, dtype=torch.float16, seed=0, pad=(0, 0), scale=1.0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    pages = [-(-n // P) for n in lens]
    N = sum(pages) + 2
    indices = torch.randperm(N, generator=gen, device=DEV)[:sum(pages)].to(torch.int32)
    starts, at = [0], [pad[0]]
    for p, n in zip(pages, news):
        starts.append(starts[-1] + p)
        at.append(at[-1] + n)
    last = [n - P * (p - 1) if p else 0 for n, p in zip(lens, pages)]
    T = at[-1] + pad[1]
    q = (torch.randn((T, Hq, D), generator=gen, device=DEV) * scale).to(dtype)
    cache = torch.randn((N, 2, Hkv, P, D), generator=gen, device=DEV).to(dtype)
    return dict(q=q, at=i32(at), cache=cache, starts=i32(starts), indices=indices, last=i32(last), lens=lens, news=news)


def rows_of(c, b, h):
    P, D = c["cache"].shape[3:]
    ids = c["indices"][int(c["starts"][b]):int(c["starts"][b + 1])].long()
    return c["cache"][ids, 0, h].reshape(-1, D)[:c["lens"][b]].double()


def scores(c, b, h, causal, scale):
    """fp64 scores [n, G, len] of a sequence and kv head, -inf where hidden, and the sum of |q k| scale of each."""
    G = c["q"].shape[1] // c["cache"].shape[2]
    L, n, r = c["lens"][b], c["news"][b], int(c["at"][b])
    q, k = c["q"][r:r + n, h * G:(h + 1) * G].double(), rows_of(c, b, h)
    x = torch.einsum("ngd,ld->ngl", q, k) * scale
    size = torch.einsum("ngd,ld->ngl", q.abs(), k.abs()) * scale
    if causal:
        pos = L - n + torch.arange(n, device=DEV)
        x = x.masked_fill((torch.arange(L, device=DEV) > pos[:, None])[:, None], -math.inf)
    return x, size


def reference_lse(c, causal, scale):
    T, Hq = c["q"].shape[:2]
    Hkv = c["cache"].shape[2]
    G = Hq // Hkv
    lse = torch.full((T, Hq), -math.inf, device=DEV)
    for b, n in enumerate(c["news"]):
        for h in range(Hkv):
            if n and c["lens"][b]:
                r = int(c["at"][b])
                lse[r:r + n, h * G:(h + 1) * G] = scores(c, b, h, causal, scale)[0].logsumexp(-1).float()
    return lse


def expect(c, lse, causal, scale, start):
    """The sums in fp64, and how far fp32 may be off.  A weight exp(x - lse): its exponent is off by at most
    (D + 4) 2^-24 of the sum of the products' sizes (the product's sums in fp32), and 4 roundings of |lse| and |x|;
    the exponential by 2^-22; the sum over r rows by r 2^-24 (all terms positive)."""
    D, Hkv = c["q"].shape[2], c["cache"].shape[2]
    G = c["q"].shape[1] // Hkv
    want, far = start.double().clone(), torch.zeros_like(start, dtype=torch.float64)
    for b, n in enumerate(c["news"]):
        L, r = c["lens"][b], int(c["at"][b])
        for h in range(Hkv):
            if not n or not L:
                continue
            x, size = scores(c, b, h, causal, scale)
            z = lse[r:r + n, h * G:(h + 1) * G].double()[..., None]
            w = torch.where(z == -math.inf, 0.0, torch.exp(x - z))
            off = (D + 4) * 2.0 ** -24 * size + 4 * 2.0 ** -24 * (z.abs() + size) + 2.0 ** -22
            want[b, h, :L] += w.sum((0, 1))
            far[b, h, :L] += torch.where(w > 0, w * off, 0.0).sum((0, 1)) + (n * G + 2) * 2.0 ** -24 * w.sum((0, 1))
            # a weight below fp32's normal range may be flushed
            far[b, h, :L] += n * G * 2.0 ** -126
    return want, far + 2.0 ** -23 * want.abs()


def check(c, causal=True, scale=None, lse=None, start=None, width=None, **kw):
    D = c["q"].shape[2]
    s = 1 / math.sqrt(D) if scale is None else scale
    lse = reference_lse(c, causal, s) if lse is None else lse
    B, Hkv, L = len(c["lens"]), c["cache"].shape[2], width or max(c["lens"] + [1])
    start = torch.rand((B, Hkv, L), device=DEV) if start is None else start
    got = accumulate_attention_weights_paged(start.clone(), c["q"], c["at"], c["cache"], c["starts"], c["indices"],
                                             c["last"], lse, causal=causal, softmax_scale=scale, **kw)
    want, far = expect(c, lse, causal, s, start)
    bad = (~((got.double() - want).abs() <= far)).nonzero()  # (NaN is bad)
    assert not bad.numel(), (bad[:4].tolist(), got[tuple(bad[0])].item(), want[tuple(bad[0])].item())
    for b, n in enumerate(c["lens"]):  # places past a sequence stay as they were
        assert same(got[b, :, n:], start[b, :, n:])
    return got


CASES = [
    # lens, news, Hq, Hkv, D, P
    ([1], [1], 1, 1, 64, 1),
    ([5, 130, 257], [1, 1, 1], 8, 2, 128, 16),
    ([300, 0, 40, 513], [3, 0, 40, 5], 8, 2, 128, 16),
    ([1000, 77], [200, 77], 4, 4, 64, 20),
    ([700], [700], 12, 4, 128, 16),
    ([260, 128, 384], [130, 128, 1], 10, 2, 64, 5),
    ([900, 50], [33, 50], 128, 1, 128, 64),
    ([2000], [1111], 7, 1, 64, 128),
    ([5000], [1], 32, 8, 128, 16),
    ([100, 200, 300], [64, 65, 63], 6, 2, 128, 8),
    ([40] * 130, [1, 2] * 65, 4, 2, 64, 8),     # many sequences
    ([300, 290], [65, 64], 4, 1, 64, 7),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens,news,Hq,Hkv,D,P", CASES)
def test_against_the_definition(lens, news, Hq, Hkv, D, P, dtype, causal):
    _lib.device_status(0, clear=True)
    check(make(lens, news, Hq, Hkv, D, P, dtype), causal)
    assert _lib.device_status(0) == 0


def test_with_the_attentions_lse_the_weights_of_a_row_sum_to_one():
    c = make([513, 100, 64], [100, 1, 64], 8, 2, 128, 16)
    _, lse = flash_attention_chunk_paged_with_lse(c["q"], c["at"], c["cache"], c["starts"], c["indices"], c["last"])
    out = torch.zeros(3, 2, 600, device=DEV)
    got = accumulate_attention_weights_paged(None, c["q"], c["at"], c["cache"], c["starts"], c["indices"], c["last"], lse,
                                             out=out)
    assert got is out
    # rows times heads of a group; each weight's sum is off by less than 1e-4 of it
    want = torch.tensor(c["news"], device=DEV)[:, None] * 4.0
    assert ((out.sum(-1) - want).abs() <= 1e-4 * want).all()


@pytest.mark.parametrize("G", [28, 33, 37, 56, 65, 100, 112])
@pytest.mark.parametrize("D", [64, 128])
def test_groups_that_leave_columns_of_a_tile_empty(G, D):
    # a tile of exactly one half of tokens, after a call that leaves NaN wherever it worked
    poison = make([2048] * 20, [256] * 20, 8, 1, D, 16, seed=1)
    poison["q"].fill_(math.nan)
    lse = torch.zeros(poison["q"].shape[:2], device=DEV)
    for half in (1, 3):
        n = 128 // G * half
        c = make([300], [n], G, 1, D, 16, seed=G)
        args = poison["q"], poison["at"], poison["cache"], poison["starts"], poison["indices"], poison["last"], lse
        accumulate_attention_weights_paged(None, *args, out=torch.zeros(20, 1, 2048, device=DEV))
        check(c)


def test_long_rows_of_few_heads_and_a_long_prompt():
    check(make([9000], [2500], 4, 1, 128, 16, seed=3))
    check(make([9000, 12000], [1, 3], 4, 1, 64, 16, torch.bfloat16, seed=4))


def test_scale_large_scores_and_padding_rows():
    c = make([300, 200], [20, 200], 4, 2, 64, 16, seed=5, pad=(3, 9), scale=8.0)
    c["q"][:3] = math.nan  # rows of no sequence
    c["q"][-9:] = math.inf
    check(c)
    check(make([300, 200], [20, 200], 4, 2, 128, 16, torch.bfloat16, seed=6), scale=0.7)


def test_rows_whose_lse_is_minus_infinity_add_nothing():
    c = make([100], [70], 4, 1, 64, 16, seed=7)
    lse = reference_lse(c, True, 0.125)
    lse[::3] = -math.inf
    check(c, lse=lse)


def test_chunk_longer_than_its_sequence():
    c = make([40, 30], [100, 30], 2, 1, 64, 16, seed=8)
    check(c)


def test_values_behind_the_mask_do_not_reach_others():
    c = make([100, 120], [10, 120], 2, 1, 64, 16, seed=9)
    clean = check(c)
    lse = reference_lse(c, True, 0.125)
    # a last page's rows behind the sequence, a hidden key and other sequences' queries
    ids = c["indices"].long()
    c["cache"][ids[6], 0, :, 4:] = math.nan
    got = check(c, lse=lse)
    assert torch.isfinite(got).all() and torch.isfinite(clean).all()
    c["q"][0] = math.nan  # a row of the first sequence: its keys, not the second's
    got = accumulate_attention_weights_paged(torch.zeros(2, 1, 120, device=DEV), c["q"], c["at"], c["cache"], c["starts"],
                                             c["indices"], c["last"], lse)
    assert torch.isfinite(got[1]).all() and torch.isnan(got[0, :, :91]).all()
    assert torch.isfinite(got[0, :, 91:]).all()  # keys that the row does not see


@pytest.mark.parametrize("form", ["wide", "odd", "dim", "heads"])
def test_strides(form):
    c = make([150, 90], [30, 2], 4, 2, 64, 16, seed=10)
    want = check(c, start=torch.zeros(2, 2, 150, device=DEV))
    q, cache = c["q"], c["cache"]
    T, Hq, D = q.shape
    if form == "wide":
        big = torch.zeros(T, Hq + 4, D + 16, dtype=q.dtype, device=DEV)
        big[:, 2:2 + Hq, 8:72] = q
        c["q"] = big[:, 2:2 + Hq, 8:72]
        pool = torch.zeros(*cache.shape[:-1], 80, dtype=q.dtype, device=DEV)
        pool[..., 8:72] = cache
        c["cache"] = pool[..., 8:72]
    elif form == "odd":
        big = torch.zeros(T, Hq, D + 3, dtype=q.dtype, device=DEV)
        big[..., 1:65] = q
        c["q"] = big[..., 1:65]
        pool = torch.zeros(*cache.shape[:-1], 67, dtype=q.dtype, device=DEV)
        pool[..., 1:65] = cache
        c["cache"] = pool[..., 1:65]
    elif form == "dim":
        c["q"] = q.transpose(1, 2).contiguous().transpose(1, 2)
        c["cache"] = cache.transpose(3, 4).contiguous().transpose(3, 4)
    else:
        c["cache"] = cache.transpose(2, 3).contiguous().transpose(2, 3)
    wide = torch.zeros(2, 4, 200, device=DEV)
    got = accumulate_attention_weights_paged(wide[:, 1:3, 7:157], c["q"], c["at"], c["cache"], c["starts"], c["indices"],
                                             c["last"], reference_lse(c, True, 0.125).t().contiguous().t())
    assert same(got, want)
    assert wide[:, 0].abs().sum() == 0 and wide[:, :, :7].abs().sum() == 0 and wide[:, :, 157:].abs().sum() == 0


def test_out_and_repeats_are_the_same():
    c = make([700, 333, 1200], [150, 333, 1], 8, 2, 128, 16, seed=11)
    lse = reference_lse(c, True, 128 ** -0.5)
    start = torch.rand(3, 2, 1200, device=DEV)
    args = (c["q"], c["at"], c["cache"], c["starts"], c["indices"], c["last"], lse)
    out = torch.full_like(start, 5.0)
    assert accumulate_attention_weights_paged(start, *args, out=out) is out
    for b, n in enumerate(c["lens"]):
        assert (out[b, :, n:] == 5).all()
    again = accumulate_attention_weights_paged(start.clone(), *args)
    for b, n in enumerate(c["lens"]):
        assert same(again[b, :, :n], out[b, :, :n])
        assert same(again[b, :, n:], start[b, :, n:])


def test_bad_tables_are_recorded():
    base = dict(lens=[100, 60], news=[10, 20], Hq=2, Hkv=1, D=64, P=16)
    for what, status in (("page", 2), ("rows", 4), ("bounds", 4), ("width", 3)):
        c = make(**base, seed=12)
        lse = reference_lse(c, True, 0.125)
        width = 100
        args = dict(at=c["at"].clone(), starts=c["starts"].clone(), indices=c["indices"].clone())
        if what == "page":
            args["indices"][8] = c["cache"].shape[0] + 3
        if what == "rows":
            args["at"][2] = 31
        if what == "bounds":
            args["starts"][2] = 50
        if what == "width":
            width = 70
        _lib.device_status(0, clear=True)
        got = accumulate_attention_weights_paged(torch.zeros(2, 1, width, device=DEV), c["q"], args["at"], c["cache"],
                                                 args["starts"], args["indices"], c["last"], lse)
        assert _lib.device_status(0, clear=True) == status, what
        want, far = expect(c, lse, True, 0.125, torch.zeros(2, 1, 100, device=DEV))
        assert ((got[0].double() - want[0, :, :width]).abs() <= far[0, :, :width]).all(), what
        if what in ("rows", "bounds"):
            assert (got[1] == 0).all()


def test_no_rows_and_no_sequences():
    c = make([20, 30], [0, 0], 2, 1, 64, 16)
    start = torch.rand(2, 1, 30, device=DEV)
    out = torch.zeros_like(start)
    accumulate_attention_weights_paged(start, c["q"], c["at"], c["cache"], c["starts"], c["indices"], c["last"],
                                       torch.zeros(0, 2, device=DEV), out=out)
    assert same(out[1], start[1]) and same(out[0, :, :20], start[0, :, :20]) and (out[0, :, 20:] == 0).all()
    e = torch.zeros(0, 1, 4, device=DEV)
    accumulate_attention_weights_paged(e, c["q"], i32([0]), c["cache"], i32([0]), i32([]), i32([]),
                                       torch.zeros(0, 2, device=DEV))


def test_graph_and_another_stream():
    c = make([400, 300], [1, 150], 8, 2, 128, 16, seed=13)
    lse = reference_lse(c, True, 128 ** -0.5)
    args = (c["q"], c["at"], c["cache"], c["starts"], c["indices"], c["last"], lse)
    start = torch.rand(2, 2, 400, device=DEV)
    want = accumulate_attention_weights_paged(start.clone(), *args)
    side, w = torch.cuda.Stream(), start.clone()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        accumulate_attention_weights_paged(w, *args)
    torch.cuda.current_stream().wait_stream(side)
    assert same(w, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        accumulate_attention_weights_paged(w, *args)
    for _ in range(2):
        w.copy_(start)
        graph.replay()
        assert same(w, want)

"""Attention behind shared prefixes against the definition in 64 bits."""
import math

import pytest
import torch

from test_paged_chunk_gpu import BF16, DEV, FP16, Case

from attention_kernel_triton_b200 import _lib
from attention_kernel_triton_b200.paged_chunk_attention import flash_attention_chunk_paged_with_lse
from attention_kernel_triton_b200.paged_kv_pages import fork_paged_kv_cache
from attention_kernel_triton_b200.paged_prefix_attention import (flash_attention_shared_prefix_paged,
                                                                 flash_attention_shared_prefix_paged_with_lse,
                                                                 shared_prefix_pages, shared_prefix_paged_into)

pytestmark = pytest.mark.gpu


def same(a, b):
    return bool(torch.equal(a, b))


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.fixture(autouse=True)
def device_status_clean():
    _lib.device_status(0, clear=True)
    yield


class Family(Case):
    """Groups (shared pages, [own tokens], [new tokens]): each sequence is the group's shared pages, then its own."""

    def __init__(self, groups, Hkv=2, G=4, D=128, P=16, dtype=FP16, seed=0, extra=2, std=1.0):
        g = torch.Generator(device=DEV).manual_seed(seed)
        cpu = torch.Generator().manual_seed(seed)
        self.Hkv, self.G, self.D, self.P, self.dtype = Hkv, G, D, P, dtype
        own_pages = [-(-n // P) for _, own, _ in groups for n in own]
        N = sum(s for s, _, _ in groups) + sum(own_pages) + extra
        place = torch.randperm(N, generator=cpu).tolist()
        self.pool = torch.full((N, 2, Hkv, P, D), math.nan, dtype=dtype, device=DEV)
        self.K, self.V, self.lens, self.news = [], [], [], []
        table, starts, last, at, bounds = [], [0], [], [0], [0]
        for shared, own, news in groups:
            mine = [place.pop() for _ in range(shared)]
            front = (torch.randn((2, Hkv, shared * P, D), generator=g, device=DEV) * std).to(dtype)
            if shared:
                self.pool[mine] = front.view(2, Hkv, shared, P, D).permute(2, 0, 1, 3, 4)
            for n, new in zip(own, news):
                k = -(-n // P)
                pages = [place.pop() for _ in range(k)]
                kv = (torch.randn((2, Hkv, k * P, D), generator=g, device=DEV) * std).to(dtype)
                kv[:, :, n:] = math.nan
                if k:
                    self.pool[pages] = kv.view(2, Hkv, k, P, D).permute(2, 0, 1, 3, 4)
                table += mine + pages
                starts.append(len(table))
                last.append(n - P * (k - 1) if k else (P if shared else 0))
                self.lens.append(shared * P + n)
                self.news.append(new)
                at.append(at[-1] + new)
                self.K.append(torch.cat((front[0], kv[0, :, :n]), 1))
                self.V.append(torch.cat((front[1], kv[1, :, :n]), 1))
            bounds.append(len(self.lens))
        self.indptr, self.indices, self.last, self.at = i32(starts), i32(table), i32(last), i32(at)
        self.bounds, self.shared = i32(bounds), i32([s for s, _, _ in groups])
        self.q = (torch.randn((at[-1], Hkv * G, D), generator=g, device=DEV) * std).to(dtype)

    def run(self, causal, scale=None, bounds=None, shared=None):
        return flash_attention_shared_prefix_paged_with_lse(
            *self.args(), self.bounds if bounds is None else bounds, self.shared if shared is None else shared,
            causal=causal, softmax_scale=scale)

    def check(self, causal, scale=None, bounds=None, shared=None):
        got, lse = self.run(causal, scale, bounds, shared)
        self.close(got, lse, causal, scale)
        assert _lib.device_status(0) == 0
        return got, lse


GROUPS = [
    (9, [1, 17, 40, 128, 129], [1, 1, 3, 60, 129]),
    (0, [33, 5], [2, 5]),
    (20, [300], [7]),
    (8, [16, 0, 32], [4, 0, 1]),
    (33, [5, 700, 64, 1, 1, 90], [5, 1, 64, 1, 0, 2]),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype,D", [(FP16, 128), (BF16, 128), (FP16, 64), (BF16, 64)])
@pytest.mark.parametrize("G,Hkv", [(1, 3), (4, 2), (8, 1)])
def test_matches_formula(G, Hkv, dtype, D, causal):
    Family(GROUPS, Hkv=Hkv, G=G, D=D, dtype=dtype, seed=G).check(causal)


@pytest.mark.parametrize("P", [1, 5, 8, 20, 48, 64, 128, 256])
@pytest.mark.parametrize("dtype,D", [(BF16, 128), (FP16, 64)])
def test_page_sizes(P, dtype, D):
    c = Family([(300 // P + 1, [1, 70, 257], [1, 3, 130]), (1, [9, 9], [1, 9])], P=P, D=D, dtype=dtype, seed=P)
    for causal in (True, False):
        c.check(causal)


@pytest.mark.parametrize("G", [3, 5, 7, 16, 48, 128])
def test_odd_groups_of_heads(G):
    Family([(12, [50, 3, 20], [40, 1, 2]), (7, [1, 1], [1, 1])], Hkv=1 + G % 2, G=G, D=64 if G == 48 else 128, dtype=BF16,
           seed=G).check(True)


def test_one_token_of_many_samples_behind_a_long_prefix():
    Family([(256, [1 + 7 * i for i in range(48)], [1] * 48)], Hkv=2, G=4, P=16, seed=1).check(True)
    Family([(40, [1 + i % 9 for i in range(150)], [1 + i % 2 for i in range(150)])], Hkv=1, G=8, P=16, seed=2).check(True)
    Family([(500, [3, 9], [1, 1])], Hkv=1, G=1, P=16, seed=3).check(True)  # few rows: units in many parts


def test_prompts_behind_documents():
    Family([(100, [260, 517], [260, 500]), (30, [130, 900, 77], [130, 129, 77])], Hkv=2, G=4, D=64, P=20, dtype=BF16,
           seed=4).check(True)
    Family([(60, [1100, 513], [1100, 400])], Hkv=1, G=2, D=128, P=16, seed=5).check(True)


def test_borders_of_the_warp_level_units():
    Family([(4, [2047, 2048, 2049, 2050], [1, 8, 8, 9])], Hkv=2, G=4, seed=20).check(True)
    Family([(4, [31, 32, 33, 2047], [31, 32, 33, 2])], Hkv=1, G=1, D=64, dtype=BF16, seed=21).check(True)
    Family([(2, [5, 16, 40, 7], [1, 2, 4, 3])], Hkv=2, G=8, D=64, seed=22).check(True)
    Family([(2, [5, 16, 40, 7], [1, 2, 4, 3])], Hkv=1, G=7, seed=23).check(False)


def test_more_sequences_than_are_ordered():
    Family([(3, [1 + i % 5 for i in range(1100)], [1] * 1100)], Hkv=1, G=2, D=64, seed=24).check(True)


def test_rows_that_a_kernel_of_their_own_joins():
    Family([(20, [700, 600], [700, 600]), (3, [33], [33])], Hkv=4, G=8, D=64, seed=25).check(True)


def test_a_long_sequence_without_a_prefix_beside_a_group():
    Family([(0, [9000], [1]), (40, [3, 5], [1, 1]), (0, [5000], [3])], Hkv=2, G=4, seed=26).check(True)


def test_scale_and_large_scores():
    Family([(9, [30, 31], [3, 4])], D=64, seed=6, std=2.0).check(True, scale=0.3)


def test_the_claim_is_cut_to_what_the_sequences_have_and_see():
    c = Family([(8, [1, 20, 3], [1, 20, 2])], seed=7)
    c.check(True, shared=i32([0]))
    c.check(True, shared=i32([5]))
    # claimed whole, though the rows of the second reach back into the shared pages
    c = Family([(8, [2, 2], [1, 40])], seed=8)
    c.check(True)
    c.check(False)
    c = Family([(8, [0, 0], [1, 2])], seed=9)  # nothing of their own
    c.check(True)
    c.check(False, shared=i32([100]))
    c.check(False, shared=i32([-4]))


def test_sequences_outside_all_groups():
    c = Family([(0, [40], [2]), (6, [9, 10], [1, 3]), (0, [77], [5])], seed=10)
    c.check(True, bounds=i32([1, 3]), shared=i32([6]))
    c.check(True, bounds=i32([0, 0, 1, 3, 3, 4]), shared=i32([3, 0, 6, 1, 2]))
    c.check(True, bounds=i32([2]), shared=i32([]))


def test_pages_in_common_are_found():
    c = Family(GROUPS, seed=11)
    full = [9, 0, 0, 8, 33]
    assert shared_prefix_pages(c.bounds, c.indptr, c.indices, c.last, 16).tolist() == full
    got, lse = flash_attention_shared_prefix_paged_with_lse(*c.args(), c.bounds)
    want, ref = c.run(True)
    assert same(got, want) and same(lse, ref)
    assert same(flash_attention_shared_prefix_paged(*c.args(), c.bounds, causal=False), c.run(False)[0])
    # a partly filled last page does not count, though both name it
    starts, table = i32([0, 3, 6, 10]), i32([4, 7, 5, 4, 7, 5, 4, 7, 5, 2])
    assert shared_prefix_pages(i32([0, 2, 3]), starts, table, i32([3, 3, 1]), 16).tolist() == [2, 0]
    assert shared_prefix_pages(i32([0, 3]), starts, table, i32([16, 16, 1]), 16).tolist() == [3]
    assert shared_prefix_pages(i32([0, 3]), starts, table, i32([16, 2, 1]), 16).tolist() == [2]


def test_with_a_forks_table():
    c = Case([150, 90], [1, 1], seed=12, extra=20)
    parents = i32([0, 0, 0, 1, 1])
    starts, table, last = fork_paged_kv_cache(c.pool, c.indptr, c.indices, c.last, parents, max_entries=3 * 10 + 2 * 6)
    c.lens, c.news = [150] * 3 + [90] * 2, [2] * 5
    c.K, c.V = [c.K[i] for i in (0, 0, 0, 1, 1)], [c.V[i] for i in (0, 0, 0, 1, 1)]
    c.indptr, c.indices, c.last, c.at = starts, table, last, i32([0, 2, 4, 6, 8, 10])
    c.q = torch.randn(10, 8, 128, device=DEV).half()
    groups = i32([0, 3, 5])
    assert shared_prefix_pages(groups, starts, table, last, 16).tolist() == [9, 5]
    got, lse = flash_attention_shared_prefix_paged_with_lse(*c.args(), groups)
    c.close(got, lse, True)


def test_rows_of_no_sequence_are_zeros():
    c = Family([(9, [20, 20], [3, 4]), (3, [5], [2])], seed=13)
    want, ref = c.run(True)
    T = c.q.shape[0]
    q = torch.full((T + 7, *c.q.shape[1:]), math.nan, dtype=c.dtype, device=DEV)
    q[3:3 + T] = c.q
    c.q, c.at = q, c.at + 3
    got, lse = c.run(True)
    assert same(got[3:3 + T], want) and same(lse[3:3 + T], ref)
    for part in (slice(0, 3), slice(3 + T, None)):
        assert (got[part] == 0).all() and (lse[part] == -math.inf).all()


def test_bad_tables_are_recorded_and_the_others_stand():
    base = Family([(9, [20, 21, 22], [3, 4, 5]), (4, [30, 31], [2, 2])], seed=14)
    O, ref, _, _ = base.exact(True)
    for what, status in (("groups", 4), ("rows", 4), ("pages", 4), ("id", 2)):
        c = Family([(9, [20, 21, 22], [3, 4, 5]), (4, [30, 31], [2, 2])], seed=14)
        bounds = c.bounds.clone()
        if what == "groups":
            bounds[1] = 9
        if what == "rows":
            c.at = c.at.clone()
            c.at[5] = 99
        if what == "pages":
            c.indptr = c.indptr.clone()
            c.indptr[5] = 999
        if what == "id":
            c.indices = c.indices.clone()
            c.indices[-1] = 10000
        got, lse = c.run(True, bounds=bounds)
        assert _lib.device_status(0, clear=True) == status, what
        rows = 16 if what == "groups" else 12  # the first group's, or all
        assert ((got[:rows].double() - O[:rows]).abs() <= 4e-3).all(), what  # (what they are: test_matches_formula)
        assert torch.isfinite(got[:rows]).all()
        if what == "rows":
            assert (got[14:] == 0).all() and (lse[14:] == -math.inf).all()


def test_values_behind_the_mask_stay_there():
    c = Family([(9, [20, 40], [2, 30])], seed=15)
    # the newest key and value of each sequence are not finite: only the last rows see them
    clean, _ = c.run(True)
    tab, starts = c.indices.tolist(), c.indptr.tolist()
    for b, n in enumerate(c.lens):
        page = tab[starts[b] + (n - 1) // 16]
        c.pool[page, 1, :, (n - 1) % 16] = math.inf
    got, _ = c.run(True)
    rows = [1, 31]
    keep = [i for i in range(32) if i not in rows]
    assert same(got[keep], clean[keep])
    assert (got[rows] == math.inf).all()
    c.pool[tab[3], 0, 0, 5] = math.nan  # a shared key: every row of that head
    got, lse = c.run(True)
    assert torch.isnan(got[:, :4]).all() and torch.isnan(lse[:, :4]).all()
    assert same(got[keep][:, 4:], clean[keep][:, 4:])


@pytest.mark.parametrize("form", ["wide", "odd", "heads"])
def test_strides(form):
    c = Family([(9, [20, 40], [2, 30]), (2, [7], [1])], D=64, seed=16)
    want, ref = c.run(True)
    if form == "wide":
        q = torch.zeros(c.q.shape[0], 12, 80, dtype=c.dtype, device=DEV)
        q[:, 2:10, 8:72] = c.q
        c.q = q[:, 2:10, 8:72]
        pool = torch.zeros(*c.pool.shape[:-1], 80, dtype=c.dtype, device=DEV)
        pool[..., 8:72] = c.pool
        c.pool = pool[..., 8:72]
    elif form == "odd":
        q = torch.zeros(c.q.shape[0], 8, 67, dtype=c.dtype, device=DEV)
        q[..., 1:65] = c.q
        c.q = q[..., 1:65]
    else:
        c.pool = c.pool.transpose(2, 3).contiguous().transpose(2, 3)
    out = torch.zeros(c.q.shape[0], 9, 72, dtype=c.dtype, device=DEV)
    lse = torch.zeros(9, c.q.shape[0], device=DEV)
    shared_prefix_paged_into(out[:, 1:, :64], *c.args(), c.bounds, c.shared, lse=lse[1:].t())
    assert same(out[:, 1:, :64], want) and same(lse[1:].t(), ref)
    assert (out[:, 0] == 0).all() and (out[..., 64:] == 0).all()


def test_the_same_as_without_groups_up_to_rounding_and_repeatable():
    c = Family([(100, [60, 70, 80, 90], [1, 5, 1, 2])] * 3, seed=17)
    plain, ref = flash_attention_chunk_paged_with_lse(*c.args())
    c.close(plain, ref, True)
    a, x = c.run(True)
    c.close(a, x, True)
    b, y = c.run(True)
    assert same(a, b) and same(x, y)


def test_graph_and_another_stream():
    c = Family([(40, [60, 70, 80], [1, 5, 1]), (12, [3, 4], [1, 2])], seed=18)
    want, ref = c.run(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, _ = c.run(True)
    torch.cuda.current_stream().wait_stream(side)
    assert same(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, lse = c.run(True)
        found = flash_attention_shared_prefix_paged(*c.args(), c.bounds)
    got.zero_()
    graph.replay()
    assert same(got, want) and same(lse, ref) and same(found, want)


def test_no_groups_need_no_pointers():
    c = Family([(4, [20, 40], [2, 3])], seed=27)
    out, lse = torch.empty_like(c.q), torch.empty(c.q.shape[:2], device=DEV)
    q, at, pool, indptr, indices, last = c.args()
    a = _lib.PrefixPagedArgs()
    k = a.chunk
    k.q, (k.q_stride_token, k.q_stride_head, k.q_stride_dim) = q.data_ptr(), q.stride()
    k.q_indptr, k.num_tokens, k.kv_cache, k.num_pages = at.data_ptr(), q.shape[0], pool.data_ptr(), pool.shape[0]
    (k.kv_stride_page, k.kv_stride_kv, k.kv_stride_head, k.kv_stride_token, k.kv_stride_dim) = pool.stride()
    k.kv_page_indptr, k.kv_page_indices, k.kv_last_page_len = indptr.data_ptr(), indices.data_ptr(), last.data_ptr()
    k.num_page_entries, k.out, k.lse = indices.numel(), out.data_ptr(), lse.data_ptr()
    (k.out_stride_token, k.out_stride_head, k.out_stride_dim) = out.stride()
    (k.lse_stride_token, k.lse_stride_head) = lse.stride()
    k.batch, k.num_qo_heads, k.num_kv_heads, k.page_size, k.head_dim, k.causal = 2, 8, 2, 16, 128, 1
    k.dtype, k.softmax_scale = _lib.AKT_FLOAT16, 128 ** -0.5
    L = _lib.lib()
    ws = torch.empty(L.akt_prefix_paged_workspace_size(a), dtype=torch.uint8, device=DEV)
    assert L.akt_prefix_paged(a, ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream) == _lib.AKT_OK
    c.close(out, lse, True)


def test_nothing_to_do():
    c = Family([(2, [3, 4], [0, 0])], seed=19)
    assert c.run(True)[0].shape == (0, 8, 128)
    assert shared_prefix_pages(i32([0]), i32([0]), i32([]), i32([]), 16).numel() == 0

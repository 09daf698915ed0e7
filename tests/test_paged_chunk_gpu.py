"""Chunk attention over a paged cache against the definition in 64 bits."""
import math

import pytest
import torch

from attention_kernel_triton_b200 import _lib
from attention_kernel_triton_b200 import workloads as W
from attention_kernel_triton_b200.decode_flash_attention_redundant_var_len_paged import flash_attention_decode_paged
from attention_kernel_triton_b200.paged_chunk_attention import (chunk_paged_into, flash_attention_chunk_paged,
                                                                flash_attention_chunk_paged_with_lse)

pytestmark = pytest.mark.gpu
DEV = "cuda"
FP16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(autouse=True)
def device_status_clean():
    _lib.device_status(0, clear=True)
    yield


class Case:
    """Sequences of `lens` tokens whose `news` newest are the queries, in a pool of shuffled pages; what no sequence
    holds (rows past a last token, pages of nobody) is NaN."""

    def __init__(self, lens, news, Hkv=2, G=4, D=128, P=16, dtype=FP16, seed=0, extra=2, std=1.0):
        g = torch.Generator(device=DEV)
        g.manual_seed(seed)
        self.lens, self.news, self.Hkv, self.G, self.D, self.P, self.dtype = lens, news, Hkv, G, D, P, dtype
        cpu = torch.Generator().manual_seed(seed)
        pages = [-(-n // P) for n in lens]
        N = sum(pages) + extra
        self.indices = torch.randperm(N, generator=cpu)[:sum(pages)].to(torch.int32).to(DEV)
        self.indptr = torch.tensor([0, *torch.tensor(pages).cumsum(0).tolist()], dtype=torch.int32, device=DEV)
        self.last = torch.tensor([n - P * (p - 1) if p else 0 for n, p in zip(lens, pages)], dtype=torch.int32, device=DEV)
        self.at = torch.tensor([0, *torch.tensor(news).cumsum(0).tolist()], dtype=torch.int32, device=DEV)
        self.pool = torch.full((N, 2, Hkv, P, D), math.nan, dtype=dtype, device=DEV)
        self.K, self.V = [], []
        ind = self.indptr.tolist()
        for b, n in enumerate(lens):
            kv = (torch.randn((2, Hkv, pages[b] * P, D), generator=g, device=DEV) * std).to(dtype)
            kv[:, :, n:] = math.nan
            own = self.indices[ind[b]:ind[b + 1]].long()
            self.pool[own] = kv.view(2, Hkv, pages[b], P, D).permute(2, 0, 1, 3, 4)
            self.K.append(kv[0, :, :n])
            self.V.append(kv[1, :, :n])
        self.q = (torch.randn((sum(news), Hkv * G, D), generator=g, device=DEV) * std).to(dtype)

    def args(self):
        return self.q, self.at, self.pool, self.indptr, self.indices, self.last

    def exact(self, causal, scale=None):
        """(O, lse, sum of weight * |v|, a bound on the scores' rounding) in 64 bits."""
        scale = scale or 1 / math.sqrt(self.D)
        O = torch.zeros(self.q.shape, dtype=torch.float64, device=DEV)
        A, S = O.clone(), torch.zeros(self.q.shape[:2], dtype=torch.float64, device=DEV)
        lse = torch.full(self.q.shape[:2], -math.inf, dtype=torch.float64, device=DEV)
        r = 0
        for b, (n, L) in enumerate(zip(self.news, self.lens)):
            if n and L:
                q = self.q[r:r + n].double().view(n, self.Hkv, self.G, self.D)
                K, V = self.K[b].double(), self.V[b].double()
                x = torch.einsum("nhgd,hld->nhgl", q, K) * scale
                size = torch.einsum("nhgd,hld->nhgl", q.abs(), K.abs()).amax(-1) * scale
                if causal:
                    pos = L - n + torch.arange(n, device=DEV)
                    hidden = torch.arange(L, device=DEV)[None] > pos[:, None]
                    x = x.masked_fill(hidden[:, None, None], -math.inf)
                z = torch.logsumexp(x, -1)
                w = torch.where(z[..., None] == -math.inf, 0.0, torch.exp(x - z[..., None].clamp(min=-1e300)))
                O[r:r + n] = torch.einsum("nhgl,hld->nhgd", w, V).flatten(1, 2)
                A[r:r + n] = torch.einsum("nhgl,hld->nhgd", w, V.abs()).flatten(1, 2)
                S[r:r + n] = size.flatten(1)
                lse[r:r + n] = z.flatten(1)
            r += n
        return O, lse, A, S

    def check(self, causal, scale=None, **kw):
        got, lse = flash_attention_chunk_paged_with_lse(*self.args(), causal=causal, softmax_scale=scale, **kw)
        self.close(got, lse, causal, scale)
        assert _lib.device_status(0) == 0
        return got, lse

    def close(self, got, lse, causal, scale=None):
        O, ref, A, S = self.exact(causal, scale)
        unit = torch.finfo(self.dtype).eps / 2
        # a score is a sum of D fp32 products, scaled: at most (D + 4) 2^-24 of the magnitudes' sum off, and so is a
        # weight, relatively (2^-20 more for the exponential and the sums of weights); the weights are rounded to the
        # type once (unit), below fp16's normal range by 2^-25 of the row's largest; then the output is rounded
        off = (self.D + 4) * 2.0 ** -24 * S + 2.0 ** -20
        tiny = 2.0 ** -25 * max([v.shape[1] * v.abs().max().item() for v in self.V if v.numel()] + [0.0])
        bound = (unit + 2 * off)[..., None] * A + unit * O.abs() + (tiny if self.dtype == FP16 else 0.0) + 2.0 ** -24
        assert torch.isfinite(got).all()
        assert ((got.double() - O).abs() <= bound).all()
        seen = torch.isfinite(ref)
        assert torch.equal(seen, torch.isfinite(lse)) and (lse[~seen] == -math.inf).all()
        assert (got[~seen] == 0).all()
        assert ((lse.double() - ref).abs()[seen] <= (off + 2.0 ** -22 * ref.abs())[seen]).all()


LENS = [1, 16, 127, 128, 129, 300, 0, 513, 40, 5]
NEWS = [1, 16, 1, 128, 60, 3, 0, 257, 0, 9]  # the last chunk is longer than its sequence


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype,D", [(FP16, 128), (BF16, 128), (FP16, 64), (BF16, 64)])
@pytest.mark.parametrize("G,Hkv", [(1, 3), (2, 2), (4, 2), (8, 1)])
def test_chunk_matches_formula(G, Hkv, dtype, D, causal):
    c = Case(LENS, NEWS, Hkv=Hkv, G=G, D=D, P=16, dtype=dtype, seed=G)
    c.check(causal)
    assert _lib.device_status(0) == 0


@pytest.mark.parametrize("P", [1, 3, 5, 8, 20, 24, 32, 40, 48, 64, 100, 128, 256, 512])
@pytest.mark.parametrize("dtype,D", [(BF16, 128), (FP16, 64)])
def test_chunk_page_sizes(P, dtype, D):
    c = Case([700, 1, P, 2 * P + 1, 131, 257], [150, 1, 1, 2, 131, 5], Hkv=2, G=4, D=D, P=P, dtype=dtype, seed=P)
    for causal in (True, False):
        c.check(causal)
    assert _lib.device_status(0) == 0


@pytest.mark.parametrize("G", [3, 5, 6, 7, 16, 48, 128])
def test_chunk_odd_groups(G):
    c = Case([333, 64, 1, 130], [100, 64, 1, 2], Hkv=1 + G % 2, G=G, D=64 if G == 48 else 128, dtype=BF16, seed=G)
    c.check(True)
    assert _lib.device_status(0) == 0


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 500])
def test_chunk_lengths_around_tiles(n):
    for L in {n, n + 1, n + 127, n + 128, 1024 + n, 1025}:
        if L >= n:
            Case([L], [n], Hkv=1, G=4, seed=n + L).check(True)
    assert _lib.device_status(0) == 0


def test_chunk_long_context_few_rows():
    # rows of few tokens whose keys are split over many CTAs
    c = Case([20011, 9000], [3, 1], Hkv=2, G=4, seed=1)
    c.check(True)
    c = Case([33000], [1], Hkv=8, G=4, D=64, dtype=BF16, seed=2)
    c.check(True)


@pytest.mark.parametrize("B", [1, 97, 300])
def test_chunk_many_sequences(B):
    lens = [(i * 37) % 400 for i in range(B)]
    news = [min(n, 1 + (i * i) % 5 if i % 7 else 70) for i, n in enumerate(lens)]
    c = Case(lens, news, Hkv=2, G=4, D=64, P=16, dtype=BF16, seed=B)
    c.check(True)
    assert _lib.device_status(0) == 0


def test_chunk_many_units_per_cta():
    # more work units than CTAs several times over: whole units first, the rest split
    c = Case([1500, 700, 2100], [1500, 300, 2000], Hkv=8, G=4, D=64, dtype=FP16, seed=3)
    c.check(True)
    c.check(False)


@pytest.mark.parametrize("new", [1, 5, 40])
def test_chunk_many_segments_and_tiles_per_cta(new):
    # each CTA walks several units of many key tiles, of one tile of rows and of two
    lens = [300 + 97 * i for i in range(64)]
    c = Case(lens, [new] * 64, Hkv=8, G=4, D=128, seed=new)
    c.check(True)
    assert _lib.device_status(0) == 0


@pytest.mark.parametrize("dtype,D", [(FP16, 128), (BF16, 64)])
def test_chunk_units_of_few_rows_among_others(dtype, D):
    # units of less than a tile of rows have the rest of their query tile cleared: at the limit, around it, after and
    # before whole tiles on the same CTA, queries apart in memory; other sequences' queries must not matter
    news = [12, 13, 1, 40, 0, 3, 70, 11] * 8
    c = Case([max(n, 200 + 53 * i) for i, n in enumerate(news)], news, Hkv=8, G=4, D=D, dtype=dtype, seed=12)
    got, lse = c.check(True)
    c.check(False)
    wide = torch.full((c.q.shape[0], 2, 32, D), math.nan, dtype=dtype, device=DEV)
    wide[:, 1] = c.q
    strided = (wide[:, 1], *c.args()[1:])
    assert torch.equal(flash_attention_chunk_paged(*strided), got)
    at = c.at.tolist()
    for b in range(0, 64, 2):  # the sequences of 13, 40, 3 and 11 tokens stay
        c.q[at[b]:at[b + 1]] = math.nan
    rest, lse2 = flash_attention_chunk_paged_with_lse(*c.args())
    for b in range(1, 64, 2):
        assert torch.equal(rest[at[b]:at[b + 1]], got[at[b]:at[b + 1]])
        assert torch.equal(lse2[at[b]:at[b + 1]], lse[at[b]:at[b + 1]])


def test_chunk_one_token_is_the_decode():
    lens = [1, 17, 500, 4000]
    c = Case(lens, [1] * 4, Hkv=2, G=4, seed=4)
    O = flash_attention_chunk_paged(*c.args())
    D = flash_attention_decode_paged(c.q.unsqueeze(2), torch.nan_to_num(c.pool), c.indptr, c.indices, c.last)
    # both round the weights and the output once; the outputs are below 4
    assert ((O - D).abs() <= 4 * 2.0 ** -10).all()


def test_chunk_large_scores_and_scale():
    c = Case([600, 90], [200, 90], G=2, std=4.0, seed=5)
    c.check(True)
    c = Case([600], [300], G=4, seed=6, dtype=BF16)
    c.check(True, scale=0.7)
    # scores that grow along the keys, so that the running maximum keeps moving
    c = Case([900], [100], Hkv=1, G=4, seed=7)
    ramp = torch.linspace(0.1, 3, 900, device=DEV)[:, None]
    c.q.fill_(0.5)
    c.K[0].copy_((ramp.expand(900, 128) * 1.0)[None].to(FP16))
    own = c.indices.long()
    k = torch.full((1, own.numel() * 16, 128), math.nan, dtype=FP16, device=DEV)
    k[:, :900] = c.K[0]
    c.pool[own, 0] = k.view(1, own.numel(), 16, 128).transpose(0, 1)
    c.check(True)


def test_chunk_nan_and_infinity_stay_behind_the_mask():
    # a token's own value row is not finite: rows before it must not change, rows from it on must be what the sum gives
    c = Case([300], [200], Hkv=2, G=4, dtype=BF16, seed=8)
    clean, lse = flash_attention_chunk_paged_with_lse(*c.args())
    for pos, value, dim in ((150, math.nan, 3), (220, math.inf, 77), (299, -math.inf, 127)):
        c.pool[int(c.indices[pos // 16]), 1, 1, pos % 16, dim] = value
    got, lse2 = flash_attention_chunk_paged_with_lse(*c.args())
    assert torch.equal(lse, lse2)
    want = clean.clone()
    want[150 - 100:, 4:, 3] = math.nan
    want[220 - 100:, 4:, 77] = math.inf
    want[299 - 100:, 4:, 127] = -math.inf
    assert torch.equal(torch.nan_to_num(got, nan=7e7), torch.nan_to_num(want, nan=7e7))
    # a key that is not finite spoils the rows that see it, and no other
    c = Case([300], [200], Hkv=1, G=4, seed=9)
    clean = flash_attention_chunk_paged(*c.args())
    c.pool[int(c.indices[250 // 16]), 0, 0, 250 % 16, 0] = math.nan
    got = flash_attention_chunk_paged(*c.args())
    assert torch.equal(got[:150], clean[:150]) and got[150:].isnan().all()


def test_chunk_strided_inputs_and_outputs():
    c = Case([200, 77], [50, 77], Hkv=2, G=4, D=64, seed=10)
    O, lse = flash_attention_chunk_paged_with_lse(*c.args())
    T = 127
    wide = torch.randn(T, 3, 8, 64, device=DEV).half()  # q inside a projection's output, heads apart
    wide[:, 1] = c.q
    q = wide[:, 1]
    out = torch.full((T, 10, 72), 5.0, dtype=FP16, device=DEV)[:, 1:9, :64]
    l2 = torch.zeros(8, T, device=DEV).t()
    chunk_paged_into(out, q, *c.args()[1:], lse=l2)
    assert torch.equal(out, O) and torch.equal(l2, lse)
    # token-major pages (heads inside a token)
    pool = c.pool.transpose(2, 3).contiguous().transpose(2, 3)
    assert torch.equal(torch.nan_to_num(flash_attention_chunk_paged(c.q, c.at, pool, *c.args()[3:])), torch.nan_to_num(O))
    # layouts that need a copy: dims apart, rows off the 16-byte grid
    qt = c.q.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(flash_attention_chunk_paged(qt, *c.args()[1:]), O)
    odd = torch.zeros(T, 8, 65, dtype=FP16, device=DEV)[:, :, 1:]
    odd.copy_(c.q)
    assert torch.equal(flash_attention_chunk_paged(odd, c.at.long(), c.pool, *c.args()[3:]), O)


def test_chunk_padding_rows_and_bad_tables():
    c = Case([50, 60], [4, 6], Hkv=2, G=2, seed=11)
    O, lse = flash_attention_chunk_paged_with_lse(*c.args())
    q = torch.cat((c.q, torch.full((5, 4, 128), math.nan, dtype=FP16, device=DEV)))  # padding of a captured batch
    O2, lse2 = flash_attention_chunk_paged_with_lse(q, *c.args()[1:])
    assert torch.equal(O2[:10], O) and (O2[10:] == 0).all() and (lse2[10:] == -math.inf).all()
    assert _lib.device_status(0) == 0
    # a page id outside the pool: its rows read as zeros, the other sequence is untouched
    bad = c.indices.clone()
    bad[1] = 1 << 20
    O2 = flash_attention_chunk_paged(c.q, c.at, c.pool, c.indptr, bad, c.last)
    assert _lib.device_status(0, clear=True) == 2
    assert torch.equal(O2[4:], O[4:]) and torch.isfinite(O2).all()
    # page bounds past the index array: the sequence counts as empty
    O2 = flash_attention_chunk_paged(c.q, c.at, c.pool, torch.tensor([0, 4, 99], dtype=torch.int32, device=DEV),
                                     c.indices, c.last)
    assert _lib.device_status(0, clear=True) == 4
    assert torch.equal(O2[:4], O[:4]) and (O2[4:] == 0).all()
    # query bounds past the rows: skipped
    flash_attention_chunk_paged(c.q, torch.tensor([0, 4, 11], dtype=torch.int32, device=DEV), *c.args()[2:])
    assert _lib.device_status(0, clear=True) == 4


def test_chunk_empty_calls():
    c = Case([0, 0], [0, 3], seed=12, extra=0)
    O, lse = flash_attention_chunk_paged_with_lse(*c.args())
    assert (O == 0).all() and (lse == -math.inf).all()
    c = Case([5], [0], seed=13)
    assert flash_attention_chunk_paged(*c.args()).shape == (0, 8, 128)
    assert _lib.device_status(0) == 0


def test_chunk_rows_do_not_depend_on_the_batch_order():
    # the same sequence alone and among others
    c = Case([700, 300, 90], [10, 300, 90], Hkv=2, G=4, seed=14)
    O = flash_attention_chunk_paged(*c.args())
    again = flash_attention_chunk_paged(*c.args())
    assert torch.equal(O, again)


def test_chunk_on_another_stream_and_in_a_graph():
    c = Case([700, 90, 33], [40, 90, 1], seed=15)
    want = flash_attention_chunk_paged(*c.args())
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    out = torch.zeros_like(c.q)
    with torch.cuda.stream(s):
        chunk_paged_into(out, *c.args())
    s.synchronize()
    assert torch.equal(out, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        chunk_paged_into(out, *c.args())
    new = torch.randn_like(c.q)
    c.q.copy_(new)
    g.replay()
    torch.cuda.synchronize()
    c.close(out, flash_attention_chunk_paged_with_lse(*c.args())[1], True)


def test_chunk_last_page_lengths_are_clamped():
    c = Case([40, 32], [8, 4], Hkv=2, G=2, seed=16)
    O = flash_attention_chunk_paged(*c.args())
    last = c.last.clone()
    last[1] = 999  # a full page of 16
    assert torch.equal(flash_attention_chunk_paged(*c.args()[:5], last), O)
    last[1] = 0  # a page that holds nothing yet: the sequence ends with the page before
    O2 = flash_attention_chunk_paged(*c.args()[:5], last)
    ref = flash_attention_chunk_paged(c.q, c.at, c.pool, torch.tensor([0, 3, 4], dtype=torch.int32, device=DEV),
                                      c.indices[:4],
                                      torch.tensor([8, 16], dtype=torch.int32, device=DEV))
    assert torch.equal(O2, ref)

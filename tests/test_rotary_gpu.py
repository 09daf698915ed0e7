"""Rotary positions against the formula in 64 bits: plain tensors (forward, inverse, gradient, in place, strided),
and fused with the append to a paged cache."""
import math

import pytest
import torch

from attention_kernel_triton_b200 import _lib
from attention_kernel_triton_b200 import workloads as W
from attention_kernel_triton_b200.paged_kv_append import append_paged_kv_cache
from attention_kernel_triton_b200.rotary_embedding import (append_rotary_paged_kv_cache, apply_rotary,
                                                           apply_rotary_qk, rotary_cos_sin, rotary_into)

pytestmark = pytest.mark.gpu
DEV = "cuda"
# half of a type's step at 1: what one rounding may move a value by, relatively
UNIT = {t: torch.finfo(t).eps / 2 for t in (torch.float16, torch.bfloat16)}


@pytest.fixture(autouse=True)
def device_status_clean():
    _lib.device_status(0, clear=True)
    yield


def turn64(x, table, positions, interleaved, inverse=False):
    """The rotation in 64 bits, and the sum of magnitudes of each output's two products."""
    R = table.shape[1]
    row = table[positions.long()].double()
    c, s = row[:, None, :R // 2], row[:, None, R // 2:]
    if inverse:
        s = -s
    x = x.double()
    y, mag = x.clone(), x.abs()
    ia = torch.arange(0, R, 2) if interleaved else torch.arange(R // 2)
    ib = ia + 1 if interleaved else ia + R // 2
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    mag[..., ia], mag[..., ib] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    return y, mag


def close(got, ref, mag):
    # two fp32 products and a sum (three roundings of 2^-24 of the magnitudes), then one rounding to the type,
    # or half of the smallest fp16 subnormal
    bound = UNIT[got.dtype] * ref.abs() + 2.0 ** -22 * mag + 2.0 ** -25
    assert torch.isfinite(got).all()
    assert ((got.double() - ref).abs() <= bound).all()


def randn(shape, dtype, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return torch.randn(shape, generator=g, device=DEV, dtype=dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,R", [(128, 128), (128, 64), (64, 64), (80, 20), (80, 32), (96, 24), (256, 256), (64, 10),
                                 (66, 66), (7, 2), (128, 2)])
def test_rotary_matches_formula(D, R, interleaved, dtype):
    T, Hq, Hkv, top = 37, 5, 2, 300
    table = rotary_cos_sin(top, R, device=DEV)
    pos = torch.randint(0, top, (T,), device=DEV, dtype=torch.int32)
    q, k = randn((T, Hq, D), dtype, 1), randn((T, Hkv, D), dtype, 2)
    for inverse in (False, True):
        q2, k2 = apply_rotary_qk(q, k, table, pos, interleaved=interleaved, inverse=inverse)
        close(q2, *turn64(q, table, pos, interleaved, inverse))
        close(k2, *turn64(k, table, pos, interleaved, inverse))
    one = apply_rotary(q, table, pos, interleaved=interleaved)
    assert torch.equal(one, apply_rotary_qk(q, k, table, pos, interleaved=interleaved)[0])
    assert torch.equal(q2[..., R:], q[..., R:])
    assert _lib.device_status(0) == 0


@pytest.mark.parametrize("T", [0, 1, 2, 255, 4097])
def test_rotary_token_counts(T):
    table = rotary_cos_sin(8192, 128, device=DEV)
    pos = torch.arange(T, device=DEV, dtype=torch.int32)
    q, k = randn((T, 3, 128), torch.bfloat16, 3), randn((T, 1, 128), torch.bfloat16, 4)
    q2, k2 = apply_rotary_qk(q, k, table, pos)
    close(q2, *turn64(q, table, pos, False))
    close(k2, *turn64(k, table, pos, False))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shift", [0, 1, 2, 4])
def test_rotary_strided_misaligned_and_in_place(shift, interleaved):
    # q, k as parts of one projection's rows whose starts and strides are off the 16-byte grid by `shift` values
    T, D, R = 19, 64, 32
    table = rotary_cos_sin(64, R, device=DEV)
    pos = torch.arange(T, device=DEV, dtype=torch.int64)  # converted
    buf = randn((T, 6 * D + 2 * shift), torch.float16, 5)
    q = buf[:, shift:shift + 4 * D].unflatten(1, (4, D))
    k = buf[:, shift + 4 * D:shift + 6 * D].unflatten(1, (2, D))
    rq, rk = turn64(q, table, pos, interleaved), turn64(k, table, pos, interleaved)
    q2, k2 = apply_rotary_qk(q, k, table, pos, interleaved=interleaved)
    close(q2, *rq)
    close(k2, *rk)
    rest = buf.clone()
    rotary_into(q, k, q, k, table, pos, interleaved=interleaved)
    assert torch.equal(q, q2) and torch.equal(k, k2)
    assert torch.equal(buf[:, :shift], rest[:, :shift])
    # a broadcast head and a transposed layout
    x = randn((T, 1, D), torch.float16, 6)
    close(apply_rotary(x.expand(T, 3, D), table, pos, interleaved=interleaved),
          *turn64(x.expand(T, 3, D), table, pos, interleaved))
    y = randn((4, D, T), torch.float16, 7).permute(2, 0, 1)
    close(apply_rotary(y, table, pos, interleaved=interleaved), *turn64(y, table, pos, interleaved))
    z = randn((4, T, D), torch.float16, 8).transpose(0, 1)
    close(apply_rotary(z, table, pos, interleaved=interleaved), *turn64(z, table, pos, interleaved))


def test_rotary_infinite_and_nan_values_stay_in_their_pairs():
    table = rotary_cos_sin(16, 64, device=DEV)
    x = torch.ones((2, 2, 64), dtype=torch.bfloat16, device=DEV)
    x[0, 0, 3], x[1, 1, 40] = math.inf, math.nan
    y = apply_rotary(x, table, torch.tensor([5, 6], dtype=torch.int32, device=DEV))
    bad = ~torch.isfinite(y)
    want = torch.zeros_like(bad)
    want[0, 0, [3, 35]] = True
    want[1, 1, [8, 40]] = True
    assert torch.equal(bad, want)


def test_rotary_positions_outside_the_table():
    table = rotary_cos_sin(10, 64, device=DEV)
    x = randn((4, 2, 128), torch.float16, 9)
    pos = torch.tensor([3, 10, -1, 9], dtype=torch.int32, device=DEV)
    y = apply_rotary(x, table, pos)
    assert (y[1:3] == 0).all()
    keep = torch.tensor([0, 3], device=DEV)
    close(y[keep], *turn64(x[keep], table, pos[keep], False))
    assert _lib.device_status(0) == 3


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_gradient(interleaved):
    T, D, R = 6, 64, 24
    table = rotary_cos_sin(100, R, device=DEV)
    pos = torch.tensor([0, 1, 99, 50, 50, 7], dtype=torch.int32, device=DEV)
    q, k = randn((T, 3, D), torch.bfloat16, 10), randn((T, 1, D), torch.bfloat16, 11)
    gq, gk = randn((T, 3, D), torch.bfloat16, 12), randn((T, 1, D), torch.bfloat16, 13)
    ql, kl = q.clone().requires_grad_(), k.clone().requires_grad_()
    q2, k2 = apply_rotary_qk(ql, kl, table, pos, interleaved=interleaved)
    dq, dk = torch.autograd.grad((q2, k2), (ql, kl), (gq, gk))
    close(dq, *turn64(gq, table, pos, interleaved, inverse=True))
    close(dk, *turn64(gk, table, pos, interleaved, inverse=True))
    (d1,) = torch.autograd.grad(apply_rotary(ql, table, pos, interleaved=interleaved), ql, gq)
    assert torch.equal(d1, dq)
    # against differences of the formula: <g, f(x + h e) - f(x)> / h, exact for a linear map
    x64 = q.double()
    for at in [(2, 1, 0), (2, 1, R // 2), (3, 0, R - 1), (4, 2, D - 1)]:
        up = x64.clone()
        up[at] += 1.0
        diff = turn64(up, table, pos, interleaved)[0] - turn64(x64, table, pos, interleaved)[0]
        want = (diff * gq.double()).sum().item()
        assert abs(dq[at].item() - want) <= UNIT[dq.dtype] * abs(want) + 2.0 ** -20 * 8
    # only one of the two is used, and its gradient is a broadcast of one value
    (dk2,) = torch.autograd.grad(apply_rotary_qk(ql, kl, table, pos, interleaved=interleaved)[1].sum(), kl)
    close(dk2, *turn64(torch.ones_like(k), table, pos, interleaved, inverse=True))


@pytest.mark.parametrize("scaling", [None, {"type": "yarn", "factor": 4.0, "original_max_positions": 64}])
@pytest.mark.parametrize("dtype,P,D,R,interleaved", [(torch.float16, 16, 128, 128, False), (torch.bfloat16, 5, 64, 64, True),
                                                     (torch.float16, 1, 64, 20, True), (torch.bfloat16, 32, 128, 24, False),
                                                     (torch.float16, 8, 66, 66, False)])
def test_append_rotary_matches_formula(dtype, P, D, R, interleaved, scaling):
    Hq, Hkv = 6, 2
    lens, new = [1, 2 * P, P + 1, 250, 40, 3], [1, 1, P, 37, 40, 0]
    indptr, indices, last, _, _, N = W.paged_layout_from_lens(lens, P, torch.Generator().manual_seed(1))
    indptr, indices, last = indptr.to(DEV), indices.to(DEV), last.to(DEV)
    app = torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()], dtype=torch.int32, device=DEV)
    T = sum(new)
    qkv = randn((T, (Hq + 2 * Hkv) * D + 3), dtype, 14)[:, :(Hq + 2 * Hkv) * D].unflatten(1, (-1, D))
    q, k, v = qkv.split((Hq, Hkv, Hkv), 1)
    table = rotary_cos_sin(256, R, scaling=scaling, device=DEV)
    pool = randn((N + 2, 2, Hkv, P, D), dtype, 15)
    before = pool.clone()
    q2 = append_rotary_paged_kv_cache(pool, q, k, v, app, indptr, indices, last, table, interleaved=interleaved)
    pos = torch.cat([torch.arange(L - n, L) for L, n in zip(lens, new)]).to(DEV)
    close(q2, *turn64(q, table, pos, interleaved))
    # the same rows through the rotation alone and the plain append: the pools agree bit for bit
    two = before.clone()
    k2 = apply_rotary(k, table, pos.int(), interleaved=interleaved)
    close(k2, *turn64(k, table, pos, interleaved))
    seq = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new))
    page = indices.cpu().long()[indptr.cpu().long()[seq] + pos.cpu() // P].to(DEV)
    two[page, 0, :, pos % P] = k2
    two[page, 1, :, pos % P] = v
    assert torch.equal(pool, two)
    if D % 8 == 0:
        three = before.clone()
        append_paged_kv_cache(three, k2, v.contiguous(), app, indptr, indices, last)
        assert torch.equal(three, pool)
    assert append_rotary_paged_kv_cache(pool, None, k, v, app, indptr, indices, last, table,
                                        interleaved=interleaved) is None
    assert torch.equal(pool, two)
    assert _lib.device_status(0) == 0


@pytest.mark.parametrize("B", [1, 31, 33, 1030])
def test_append_rotary_finds_its_sequence(B):
    # one token or none per sequence: the search over the sequences, runs of empty ones among them
    lens = [1 + i % 7 for i in range(B)]
    new = [0 if i % 3 == 1 else 1 for i in range(B)]
    indptr, indices, last, _, _, N = W.paged_layout_from_lens(lens, 4, torch.Generator().manual_seed(2))
    app = torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()], dtype=torch.int32, device=DEV)
    T = sum(new)
    x = torch.arange(1, T + 1, device=DEV, dtype=torch.float16)[:, None, None].expand(T, 1, 64).contiguous()
    table = rotary_cos_sin(8, 64, device=DEV)
    pool = torch.zeros((N, 2, 1, 4, 64), dtype=torch.float16, device=DEV)
    append_rotary_paged_kv_cache(pool, None, x, x, app, indptr.to(DEV), indices.to(DEV), last.to(DEV), table)
    want = torch.zeros((N, 4))
    t = 0
    for b in range(B):
        if new[b]:
            t += 1
            pos = lens[b] - 1
            want[int(indices[int(indptr[b]) + pos // 4]), pos % 4] = t
    assert torch.equal(pool[:, 1, 0, :, 0].float().cpu(), want)
    assert _lib.device_status(0) == 0


def test_append_rotary_bad_tables_are_recorded():
    table = rotary_cos_sin(18, 64, device=DEV)
    c = W.make_paged(B=1, Hq=4, Hkv=2, D=64, page_size=16, lens=[20], seed=4, device=DEV)
    k = torch.ones(3, 2, 64, dtype=torch.float16, device=DEV)
    q = torch.ones(3, 4, 64, dtype=torch.float16, device=DEV)
    app = torch.tensor([0, 3], dtype=torch.int32, device=DEV)
    pool = c.cache.clone()
    # positions 17, 18, 19: the last two are past the table
    q2 = append_rotary_paged_kv_cache(pool, q, k, k, app, c.indptr, c.indices, c.last_page_len, table)
    assert _lib.device_status(0, clear=True) == 3
    assert (q2[1:] == 0).all() and (q2[0] != 0).any()
    assert int((pool != c.cache).any(-1).any(-2).sum()) == 2  # K and V of one row
    table = rotary_cos_sin(32, 64, device=DEV)  # every position has its row below
    pool = c.cache.clone()
    bad = c.indices.clone()
    bad[1] = -5
    q2 = append_rotary_paged_kv_cache(pool, q, k, k, app, c.indptr, bad, c.last_page_len, table)
    assert _lib.device_status(0, clear=True) == 2
    assert torch.equal(pool, c.cache) and (q2 == 0).all()
    q2 = append_rotary_paged_kv_cache(pool, q, k, k, app, torch.tensor([0, 9], dtype=torch.int32, device=DEV),
                                      c.indices, c.last_page_len, table)
    assert _lib.device_status(0, clear=True) == 4
    assert torch.equal(pool, c.cache) and (q2 == 0).all()


def test_rotary_on_another_stream_and_in_a_graph():
    table = rotary_cos_sin(64, 64, device=DEV)
    x = randn((33, 4, 64), torch.bfloat16, 16)
    pos = torch.arange(33, device=DEV, dtype=torch.int32)
    want = apply_rotary(x, table, pos)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    out = torch.empty_like(x)
    with torch.cuda.stream(s):
        rotary_into(out, None, x, None, table, pos)
    s.synchronize()
    assert torch.equal(out, want)
    g = torch.cuda.CUDAGraph()
    out.zero_()
    with torch.cuda.graph(g):
        rotary_into(out, None, x, None, table, pos)
    x.neg_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, -want)

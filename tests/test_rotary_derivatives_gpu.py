"""Derivatives past the first, and forward mode, of the rotary calls on the GPU against the formula in 64 bits."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from attention_kernel_triton_b200.rotary_embedding import apply_rotary, apply_rotary_qk, rotary_cos_sin

pytestmark = pytest.mark.gpu
DEV = "cuda"
UNIT = {t: torch.finfo(t).eps / 2 for t in (torch.float16, torch.bfloat16)}


def turn64(x, table, positions, interleaved, inverse=False, magnitudes=False):
    """The rotation in 64 bits; with `magnitudes`, the sums of the products' magnitudes in its place."""
    R = table.shape[1]
    row = table[positions.long()].double()[:, None]
    c, s = row[..., :R // 2], row[..., R // 2:]
    s = -s if inverse else s
    y = x.double().clone()
    ia = torch.arange(0, R, 2) if interleaved else torch.arange(R // 2)
    ib = ia + 1 if interleaved else ia + R // 2
    a, b = y[..., ia].clone(), y[..., ib].clone()
    if magnitudes:
        a, b, c, s = a.abs(), b.abs(), c.abs(), -s.abs()
        y[..., ia], y[..., ib] = a * c - b * s, b * c - a * s
        return y.abs()
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    return y


def one_turn_off(x, table, pos, interleaved, inverse=False):
    """What a rotation of x may be off by: fp32 products and sum, one rounding, half of fp16's smallest step."""
    return (UNIT[x.dtype] * turn64(x, table, pos, interleaved, inverse).abs() +
            2.0 ** -22 * turn64(x, table, pos, interleaved, magnitudes=True) + 2.0 ** -25)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
def test_second_derivative(interleaved, dtype):
    # z = sum f(x)^2, g = dz/dx, h = d(g.v)/dx = f^T(2 f(v)) = 2 v: two turns and exact doublings
    D, R, T = 64, 24, 9
    table = rotary_cos_sin(100, R, device=DEV)
    pos = torch.randint(0, 100, (T,), device=DEV, dtype=torch.int32)
    gen = torch.Generator(device=DEV).manual_seed(1)
    q = torch.randn((T, 3, D), generator=gen, device=DEV, dtype=dtype).requires_grad_()
    k = torch.randn((T, 1, D), generator=gen, device=DEV, dtype=dtype).requires_grad_()
    vq, vk = torch.randn(q.shape, generator=gen, device=DEV, dtype=dtype), torch.randn(k.shape, generator=gen, device=DEV, dtype=dtype)
    y, z = apply_rotary_qk(q, k, table, pos, interleaved=interleaved)
    gq, gk = torch.autograd.grad((y * y).sum() + (z * z).sum(), (q, k), create_graph=True)
    hq, hk = torch.autograd.grad((gq, gk), (q, k), (vq, vk))
    y1 = apply_rotary(q, table, pos, interleaved=interleaved)
    (g1,) = torch.autograd.grad((y1 * y1).sum(), q, create_graph=True)
    (h1,) = torch.autograd.grad(g1, q, vq)
    assert torch.equal(h1, hq)
    for h, v in ((hq, vq), (hk, vk)):
        first = one_turn_off(v, table, pos, interleaved)
        carried = 2 * turn64(first, table, pos, interleaved, magnitudes=True)
        # the second turn's own rounding, of a value that the first's may have moved
        own = (UNIT[dtype] * (2 * v.double().abs() + carried) + 2.0 ** -25 +
               2.0 ** -22 * 2 * turn64(turn64(v, table, pos, interleaved).abs() + first, table, pos, interleaved, magnitudes=True))
        assert ((h.double() - 2 * v.double()).abs() <= carried + own).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
def test_forward_mode(interleaved, dtype):
    D, R, T = 80, 32, 11
    table = rotary_cos_sin(50, R, device=DEV)
    pos = torch.randint(0, 50, (T,), device=DEV, dtype=torch.int32)
    gen = torch.Generator(device=DEV).manual_seed(2)
    q, k, tq = (torch.randn((T, h, D), generator=gen, device=DEV, dtype=dtype) for h in (4, 2, 4))
    plain = apply_rotary_qk(q, k, table, pos, interleaved=interleaved)
    with fwAD.dual_level():
        y, z = apply_rotary_qk(fwAD.make_dual(q, tq), k, table, pos, interleaved=interleaved)
        y, t = fwAD.unpack_dual(y)
        assert torch.equal(y, plain[0]) and torch.equal(fwAD.unpack_dual(z).primal, plain[1])
        one = fwAD.unpack_dual(apply_rotary(fwAD.make_dual(q, tq), table, pos, interleaved=interleaved)).tangent
    assert t.dtype == dtype and torch.equal(t, one)
    want = turn64(tq, table, pos, interleaved)
    assert ((t.double() - want).abs() <= one_turn_off(tq, table, pos, interleaved)).all()


def test_function_transforms():
    T, D = 7, 64
    table = rotary_cos_sin(20, D, device=DEV)
    pos = torch.arange(T, device=DEV, dtype=torch.int32)
    gen = torch.Generator(device=DEV).manual_seed(3)
    q, t = (torch.randn((T, 2, D), generator=gen, device=DEV, dtype=torch.float16) for _ in range(2))
    f = lambda x: apply_rotary(x, table, pos)  # noqa: E731
    y, ty = torch.func.jvp(f, (q,), (t,))
    assert torch.equal(y, f(q)) and torch.equal(ty, f(t))
    g = torch.func.grad(lambda x: (f(x) * t).sum())(q)
    assert torch.equal(g, apply_rotary(t, table, pos, inverse=True))

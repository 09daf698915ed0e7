"""The derivative rules of the rotary calls, with the rotation's launch replaced by values that autograd does not see
(as a launch's are): gradients of gradients, forward mode, and the refusal of a table that wants a gradient."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from attention_kernel_triton_b200 import rotary_embedding as R

T, D = 5, 16


def turn(x, table, positions, interleaved, inverse):
    half = table.shape[1] // 2
    row = table[positions.long()][:, None]
    c, s = row[..., :half], row[..., half:]
    s = -s if inverse else s
    a, b = (x[..., 0:2 * half:2], x[..., 1:2 * half:2]) if interleaved else (x[..., :half], x[..., half:2 * half])
    pair = (a * c - b * s, b * c + a * s)
    turned = torch.stack(pair, -1).flatten(-2) if interleaved else torch.cat(pair, -1)
    return torch.cat((turned, x[..., 2 * half:]), -1)


@pytest.fixture(autouse=True)
def values_only(monkeypatch):
    def forward(q, k, cos_sin, positions, interleaved, inverse):
        with torch.no_grad():
            assert all(t is None or t.data_ptr() for t in (q, k, cos_sin, positions))  # a launch takes addresses
            q_out = q.new_empty(q.shape)
            q_out.data.copy_(turn(q.detach(), cos_sin, positions, interleaved, inverse))
            k_out = None if k is None else k.new_empty(k.shape)
            if k is not None:
                k_out.data.copy_(turn(k.detach(), cos_sin, positions, interleaved, inverse))
        return q_out, k_out
    monkeypatch.setattr(R, "_forward", forward)


def inputs(rotary_dim, requires_grad=True):
    g = torch.Generator().manual_seed(0)
    rand = lambda h: torch.randn((T, h, D), generator=g, dtype=torch.float64).requires_grad_(requires_grad)  # noqa: E731
    table = R.rotary_cos_sin(40, rotary_dim, device="cpu").double()
    return rand(3), rand(1), table, torch.tensor([0, 3, 39, 7, 7], dtype=torch.int32)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rotary_dim", [D, 6])
def test_first_and_second_derivatives(rotary_dim, interleaved):
    q, k, table, pos = inputs(rotary_dim)
    qk = lambda q, k: R.apply_rotary_qk(q, k, table, pos, interleaved)  # noqa: E731
    one = lambda q: R.apply_rotary(q, table, pos, interleaved, inverse=True)  # noqa: E731
    assert torch.autograd.gradcheck(qk, (q, k), check_forward_ad=True)
    assert torch.autograd.gradgradcheck(qk, (q, k))
    assert torch.autograd.gradcheck(one, (q,), check_forward_ad=True)
    assert torch.autograd.gradgradcheck(one, (q,))


def test_gradient_penalty_is_the_formula_s():
    q, k, table, pos = inputs(D)

    def penalty(f):
        y, z = f(q, k)
        grads = torch.autograd.grad((y ** 3).sum() + (z ** 4).sum(), (q, k), create_graph=True)
        return torch.autograd.grad(sum((x ** 2).sum() for x in grads) + (y * y).sum(), (q, k))

    want = penalty(lambda q, k: (turn(q, table, pos, False, False), turn(k, table, pos, False, False)))
    got = penalty(lambda q, k: R.apply_rotary_qk(q, k, table, pos))
    for a, b in zip(got, want):
        torch.testing.assert_close(a, b)


@pytest.mark.parametrize("which", ["q", "k", "both"])
def test_tangents(which):
    q, k, table, pos = inputs(10, requires_grad=False)
    tq, tk = torch.randn_like(q), torch.randn_like(k)
    with fwAD.dual_level():
        dq = fwAD.make_dual(q, tq) if which != "k" else q
        dk = fwAD.make_dual(k, tk) if which != "q" else k
        y, z = R.apply_rotary_qk(dq, dk, table, pos, interleaved=True)
        for out, t, there in ((y, tq, which != "k"), (z, tk, which != "q")):
            got = fwAD.unpack_dual(out).tangent
            if there:
                torch.testing.assert_close(got, turn(t, table, pos, True, False))
            else:
                assert got is None or not got.any()
        with torch.no_grad():
            got = fwAD.unpack_dual(R.apply_rotary(fwAD.make_dual(q, tq), table, pos)).tangent
        torch.testing.assert_close(got, turn(tq, table, pos, False, False))


def test_function_transforms():
    q, k, table, pos = inputs(D, requires_grad=False)
    t = torch.randn_like(q)
    y, ty = torch.func.jvp(lambda q: R.apply_rotary(q, table, pos), (q,), (t,))
    torch.testing.assert_close(y, turn(q, table, pos, False, False))
    torch.testing.assert_close(ty, turn(t, table, pos, False, False))
    g = torch.func.grad(lambda q: (R.apply_rotary(q, table, pos) * t).sum())(q)
    torch.testing.assert_close(g, turn(t, table, pos, False, True))


def test_a_table_that_wants_a_gradient_is_refused():
    q, k, table, pos = inputs(D)
    wants = table.clone().requires_grad_()
    for x, y in ((q, k), (q.detach(), k.detach())):
        with pytest.raises(ValueError):
            R.apply_rotary_qk(x, y, wants, pos)
        with pytest.raises(ValueError):
            R.apply_rotary(x, wants, pos)
    with torch.no_grad():  # nobody asks for one here
        R.apply_rotary_qk(q, k, wants, pos)
    with fwAD.dual_level():
        with pytest.raises(ValueError):
            R.apply_rotary(q, fwAD.make_dual(table, torch.ones_like(table)), pos)

"""Rotary positions: the table of angles, the rotation of plain tensors (with
its gradient) and the rotation fused with the append to a paged KV cache.

The reference starts from queries and keys that are already rotated; these are
the steps before it.  A model keeps one table, ``rotary_cos_sin(...)``
(``[max_positions, rotary_dim]`` fp32: the cosines of ``rotary_dim / 2`` angles,
then their sines), and hands it to every call.  Pair ``i`` of a head's first
``rotary_dim`` values, ``(x[i], x[i + rotary_dim / 2])`` or, ``interleaved``,
``(x[2i], x[2i + 1])``, becomes ``(a c - b s, b c + a s)``; the values past
``rotary_dim`` are copied.  Sums are in fp32, rounded once to the tensors' type.
Runs ``akt_rotary`` / ``akt_append_rotary_paged_kv`` (sm_100a) on torch's
current stream.
"""
from __future__ import annotations

import math

import torch
from torch.autograd import forward_ad

from . import _lib


def rotary_frequencies(rotary_dim, base=10000.0, scaling=None):
    """``(angles per position, fp64 [rotary_dim / 2]; factor on cos and sin)``.

    ``scaling`` (a dict) stretches the angles for contexts past the trained length:

    * ``{"type": "linear", "factor": f}``: every angle divided by ``f``;
    * ``{"type": "ntk", "factor": f}``: the base raised to
      ``base * f ** (rotary_dim / (rotary_dim - 2))``, which divides the slowest
      angle by ``f`` and leaves the fastest;
    * ``{"type": "yarn", "factor": f, "original_max_positions": n}`` (optional
      ``beta_fast`` 32, ``beta_slow`` 1, ``attention_factor`` ``0.1 ln f + 1``):
      angles that turn more than ``beta_fast`` times in ``n`` positions are kept,
      those that turn less than ``beta_slow`` times divided by ``f``, and the ones
      between mixed linearly over their index (Peng et al., "YaRN", 2023);
    * ``{"type": "banded", "factor": f, "original_max_positions": n,
      "low_freq_factor": a, "high_freq_factor": b}``: by wave length ``w = 2 pi /
      angle``: kept below ``n / b``, divided by ``f`` above ``n / a``, between them
      mixed linearly in ``n / w``.
    """
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError("rotary_dim must be positive and even")
    if not base > 0:
        raise ValueError("base must be positive")
    i = torch.arange(rotary_dim // 2, dtype=torch.float64)
    freq = float(base) ** (-2 * i / rotary_dim)
    if scaling is None:
        return freq, 1.0
    kind = scaling.get("type")
    f = float(scaling["factor"])
    if not f > 0:
        raise ValueError("scaling factor must be positive")
    if kind == "linear":
        return freq / f, 1.0
    if kind == "ntk":
        if rotary_dim == 2:
            raise ValueError("ntk scaling needs rotary_dim > 2")
        return (float(base) * f ** (rotary_dim / (rotary_dim - 2))) ** (-2 * i / rotary_dim), 1.0
    if kind == "yarn":
        n = float(scaling["original_max_positions"])

        def index_of(turns):  # index of the angle that makes so many turns in n positions
            return rotary_dim * math.log(n / (turns * 2 * math.pi)) / (2 * math.log(base))

        lo = max(math.floor(index_of(float(scaling.get("beta_fast", 32.0)))), 0)
        hi = min(math.ceil(index_of(float(scaling.get("beta_slow", 1.0)))), rotary_dim - 1)
        ramp = ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        default = 0.1 * math.log(f) + 1.0 if f > 1 else 1.0
        return freq / f * ramp + freq * (1 - ramp), float(scaling.get("attention_factor", default))
    if kind == "banded":
        n = float(scaling["original_max_positions"])
        a, b = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
        if not b > a:
            raise ValueError("high_freq_factor must exceed low_freq_factor")
        keep = ((n * freq / (2 * math.pi) - a) / (b - a)).clamp(0, 1)
        return freq * keep + freq / f * (1 - keep), 1.0
    raise ValueError(f"unknown rotary scaling {kind!r}")


def rotary_cos_sin(max_positions, rotary_dim, base=10000.0, scaling=None, device="cuda"):
    """The table ``[max_positions, rotary_dim]`` (fp32) for the calls below, built once:
    angles in fp64 (an fp32 product is off by 0.008 at position 131072), rounded at the end."""
    freq, factor = rotary_frequencies(rotary_dim, base, scaling)
    angle = torch.arange(max_positions, dtype=torch.float64)[:, None] * freq
    return torch.cat((angle.cos() * factor, angle.sin() * factor), 1).float().to(device)


_rotary = _lib.Entry("akt_rotary", _lib.RotaryArgs, _lib.c_void_p)
_append_rotary = _lib.Entry("akt_append_rotary_paged_kv", _lib.AppendRotaryArgs, _lib.c_void_p)


def _check_table(cos_sin, D):
    if cos_sin.dim() != 2 or cos_sin.dtype is not torch.float32:
        raise ValueError("cos_sin must be fp32 [max_positions, rotary_dim] on the tensors' device")
    R = cos_sin.shape[1]
    if R % 2 or R > D:
        raise ValueError("rotary_dim (the table's width) must be even and at most the head dim")
    return cos_sin if cos_sin.stride(1) == 1 and cos_sin.stride(0) >= R else cos_sin.contiguous()


def _unit(x):
    return x if x.stride(-1) == 1 else x.contiguous()


def rotary_into(q_out, k_out, q, k, cos_sin, positions, interleaved=False, inverse=False):
    """Rotate ``q [T, Hq, D]`` into ``q_out`` and, unless ``k`` is None, ``k [T, Hkv, D]``
    into ``k_out`` (either may be its input: in place)."""
    shape = q.shape
    if len(shape) != 3 or q_out.shape != shape:
        raise ValueError("tensors must be [tokens, heads, head_dim], an output of its input's shape")
    T, Hq, D = shape
    if k is None:
        index = _lib.device_index(q, q_out, cos_sin)
        kp, Hkv = (0, 0, 0, 0, 0, 0, 0, 0), 0
    else:
        index = _lib.device_index(q, q_out, k, k_out, cos_sin)
        ks = k.shape
        if len(ks) != 3 or ks[0] != T or ks[2] != D or k_out.shape != ks:
            raise ValueError("q and k must be [tokens, heads, head_dim] with the same tokens and head_dim")
        if not (k.dtype == k_out.dtype == q.dtype):
            raise TypeError("q, k and the outputs must share one dtype")
        k = _unit(k)
        kp, Hkv = (k.data_ptr(), *k.stride(), k_out.data_ptr(), *k_out.stride()), ks[1]
    if q_out.dtype != q.dtype:
        raise TypeError("q, k and the outputs must share one dtype")
    table = _check_table(cos_sin, D)
    pos = _lib.list_i32(positions, q)
    if pos.dim() != 1 or pos.shape[0] != T:
        raise ValueError("positions must hold one position per token")
    q = _unit(q)
    top, R = table.shape
    values = (q.data_ptr(), *q.stride(), *kp[:4], q_out.data_ptr(), *q_out.stride(), *kp[4:], table.data_ptr(),
              table.stride(0), top, pos.data_ptr(), T, Hq, Hkv, D, R, bool(interleaved), bool(inverse),
              _lib.dtype_code(q))
    with _lib.on_index(index):
        rc = _rotary(values, _lib.raw_stream(index))
        if rc:
            _lib.check(rc)
    return q_out, k_out


def _forward(q, k, cos_sin, positions, interleaved, inverse):
    q_out, k_out = q.new_empty(q.shape), None if k is None else k.new_empty(k.shape)
    return rotary_into(q_out, k_out, q, k, cos_sin, positions, interleaved, inverse)


class _Rotary(torch.autograd.Function):
    """The rotation is linear and orthogonal: its tangent is the same turn, its gradient the inverse
    one.  Both rules apply the function itself, so that derivatives of every order have theirs."""

    @staticmethod
    def forward(q, k, cos_sin, positions, interleaved, inverse):
        return _forward(q, k, cos_sin, positions, interleaved, inverse)

    @staticmethod
    def setup_context(ctx, inputs, output):
        _, _, cos_sin, positions, interleaved, inverse = inputs
        ctx.save_for_backward(cos_sin, positions)
        ctx.save_for_forward(cos_sin, positions)
        ctx.how = interleaved, inverse

    @staticmethod
    def backward(ctx, dq, dk):
        interleaved, inverse = ctx.how
        return *_Rotary.apply(dq, dk, *ctx.saved_tensors, interleaved, not inverse), None, None, None, None

    @staticmethod
    def jvp(ctx, tq, tk, *_):
        return _Rotary.apply(tq, tk, *ctx.saved_tensors, *ctx.how)


class _RotaryOne(torch.autograd.Function):
    """``_Rotary`` for one tensor."""

    @staticmethod
    def forward(x, cos_sin, positions, interleaved, inverse):
        return _forward(x, None, cos_sin, positions, interleaved, inverse)[0]

    @staticmethod
    def setup_context(ctx, inputs, output):
        _, cos_sin, positions, interleaved, inverse = inputs
        ctx.save_for_backward(cos_sin, positions)
        ctx.save_for_forward(cos_sin, positions)
        ctx.how = interleaved, inverse

    @staticmethod
    def backward(ctx, dx):
        interleaved, inverse = ctx.how
        return _RotaryOne.apply(dx, *ctx.saved_tensors, interleaved, not inverse), None, None, None, None

    @staticmethod
    def jvp(ctx, tx, *_):
        return _RotaryOne.apply(tx, *ctx.saved_tensors, *ctx.how)


def _differentiated(cos_sin, q, k):
    """Whether a derivative in q or k (or None) is asked for, backward or forward; the table has none."""
    of_table = of_rows = False
    if torch.is_grad_enabled():
        of_table, of_rows = cos_sin.requires_grad, q.requires_grad or k is not None and k.requires_grad
    if getattr(forward_ad, "_current_level", 0) >= 0:  # (a tangent lives inside a dual level only)
        def moves(t):
            return t is not None and forward_ad.unpack_dual(t).tangent is not None
        of_table, of_rows = of_table or moves(cos_sin), of_rows or moves(q) or moves(k)
    if of_table:
        raise ValueError("cos_sin is a constant of the rotation: it takes no gradient and no tangent")
    return of_rows


def apply_rotary_qk(q, k, cos_sin, positions, interleaved=False, inverse=False):
    """
    q: [T, Hq, D], k: [T, Hkv, D] (fp16 or bf16; any strides with unit dim stride)
    cos_sin: [max_positions, rotary_dim] (fp32), positions: [T] (int32)
    returns (q', k') of the same shapes; a position outside the table gives zeros (status 3)

    ``inverse`` turns the other way, which is the gradient too: a training step either
    calls it on the outputs' gradients or lets autograd do so (any order, and forward mode;
    a table that requires a gradient is refused).
    """
    if _differentiated(cos_sin, q, k):
        return _Rotary.apply(q, k, cos_sin, positions, interleaved, inverse)
    return _forward(q, k, cos_sin, positions, interleaved, inverse)


def apply_rotary(x, cos_sin, positions, interleaved=False, inverse=False):
    """``apply_rotary_qk`` for one tensor ``x [T, H, D]``."""
    if _differentiated(cos_sin, x, None):
        return _RotaryOne.apply(x, cos_sin, positions, interleaved, inverse)
    return _forward(x, None, cos_sin, positions, interleaved, inverse)[0]


def append_rotary_paged_kv_cache(paged_kv_cache, q, append_k, append_v, append_indptr, kv_page_indptr,
                                 kv_page_indices, kv_last_page_len, cos_sin, interleaved=False):
    """``paged_kv_append.append_paged_kv_cache`` with the keys rotated to their positions in
    their sequences on the way, and the rotated queries ``[num_append, Hq, D]`` returned.

    ``q`` (or None: nothing is returned), ``append_k`` and ``append_v`` are
    ``[num_append, heads, D]``, ragged by ``append_indptr [B + 1]``; the page table already
    describes the sequences after the append.  One pass: the rotated keys are never stored
    outside the pool.  For serving: no gradient.
    """
    index = _lib.device_index(paged_kv_cache, append_k, append_v, cos_sin)
    dtype = paged_kv_cache.dtype
    if append_k.dtype != dtype or append_v.dtype != dtype:
        raise TypeError("the pool and the appended rows must share one dtype")
    pool = paged_kv_cache.shape
    if len(pool) != 5 or pool[1] != 2:
        raise ValueError("paged_kv_cache must be [num_pages, 2, Hkv, page_size, D]")
    N, _, Hkv, P, D = pool
    shape = append_k.shape
    if len(shape) != 3 or shape[1] != Hkv or shape[2] != D or append_v.shape != shape:
        raise ValueError("append_k and append_v must be [num_append, Hkv, D]")
    T = shape[0]
    table = _check_table(cos_sin, D)
    indptr = _lib.list_i32(kv_page_indptr, append_k)
    indices = _lib.list_i32(kv_page_indices, append_k)
    last = _lib.list_i32(kv_last_page_len, append_k)
    app = _lib.list_i32(append_indptr, append_k)
    B = indptr.numel() - 1
    if app.numel() != B + 1 or last.numel() != B:
        raise ValueError("append_indptr and kv_page_indptr must have B+1 entries and kv_last_page_len B entries")
    k, v = _unit(append_k), _unit(append_v)
    q_out, qp, Hq = None, (0, 0, 0, 0, 0, 0, 0, 0), 0
    if q is not None:
        _lib.device_index(paged_kv_cache, q)
        if q.dtype != dtype:
            raise TypeError("the pool and the appended rows must share one dtype")
        if q.dim() != 3 or q.shape[0] != T or q.shape[2] != D:
            raise ValueError("q must be [num_append, Hq, D]")
        q = _unit(q)
        Hq = q.shape[1]
        q_out = q.new_empty(q.shape)
        qp = (q.data_ptr(), *q.stride(), q_out.data_ptr(), *q_out.stride())
    top, R = table.shape
    values = (paged_kv_cache.data_ptr(), *paged_kv_cache.stride(), N, indptr.data_ptr(), indices.data_ptr(),
              last.data_ptr(), indices.numel(), k.data_ptr(), *k.stride(), v.data_ptr(), *v.stride(), app.data_ptr(), T,
              B, Hkv, P, D, _lib.dtype_code(k), *qp, table.data_ptr(), table.stride(0), top, Hq, R, bool(interleaved))
    with _lib.on_index(index):
        rc = _append_rotary(values, _lib.raw_stream(index))
        if rc:
            _lib.check(rc)
    return q_out

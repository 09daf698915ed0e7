"""The table of angles of the rotary positions (host, 64 bits) and what the calls refuse."""
import math

import pytest
import torch

from attention_kernel_triton_b200 import _lib
from attention_kernel_triton_b200.rotary_embedding import (append_rotary_paged_kv_cache, apply_rotary_qk,
                                                           rotary_cos_sin, rotary_frequencies)


def test_table_holds_cosines_then_sines():
    t = rotary_cos_sin(131073, 8, base=500.0, device="cpu")
    assert t.shape == (131073, 8) and t.dtype == torch.float32
    for p in (0, 1, 777, 131072):
        for i in range(4):
            a = p * 500.0 ** (-2 * i / 8)
            # the angle is exact to 2^-53 of itself, the entries are rounded to fp32 once
            assert abs(t[p, i].item() - math.cos(a)) <= 2.0 ** -25 + a * 2.0 ** -51
            assert abs(t[p, 4 + i].item() - math.sin(a)) <= 2.0 ** -25 + a * 2.0 ** -51


def test_linear_and_ntk_scaling():
    f, _ = rotary_frequencies(64)
    g, m = rotary_frequencies(64, scaling={"type": "linear", "factor": 4})
    assert torch.equal(g, f / 4) and m == 1.0
    g, m = rotary_frequencies(64, scaling={"type": "ntk", "factor": 4})
    assert m == 1.0 and g[0] == f[0]
    assert abs(g[-1] * 4 / f[-1] - 1) < 1e-12
    assert ((g <= f) & (g >= f / 4 * (1 - 1e-12))).all()


def test_yarn_scaling():
    n, f = 4096, 16.0
    base, _ = rotary_frequencies(128)
    g, m = rotary_frequencies(128, scaling={"type": "yarn", "factor": f, "original_max_positions": n})
    assert abs(m - (0.1 * math.log(16) + 1)) < 1e-12
    ratio = g / base
    # the index ranges are rounded outwards, so beyond them the ends hold exactly
    turns = base * n / (2 * math.pi)
    assert (ratio[turns > 33] == 1).all() and torch.allclose(ratio[turns < 0.8], torch.tensor(1 / f, dtype=torch.float64))
    assert (ratio.diff() <= 1e-15).all()
    _, m = rotary_frequencies(128, scaling={"type": "yarn", "factor": f, "original_max_positions": n,
                                            "attention_factor": 1.25})
    assert m == 1.25
    t = rotary_cos_sin(4, 128, scaling={"type": "yarn", "factor": f, "original_max_positions": n}, device="cpu")
    assert torch.allclose(t[0, :64], torch.full((64,), 0.1 * math.log(16) + 1))


def test_banded_scaling():
    s = {"type": "banded", "factor": 8.0, "original_max_positions": 8192, "low_freq_factor": 1.0, "high_freq_factor": 4.0}
    base, _ = rotary_frequencies(128, base=500000.0)
    g, m = rotary_frequencies(128, base=500000.0, scaling=s)
    assert m == 1.0
    for f0, f1 in zip(base.tolist(), g.tolist()):
        w = 2 * math.pi / f0
        if w < 8192 / 4:
            assert f1 == f0
        elif w > 8192:
            assert abs(f1 * 8 / f0 - 1) < 1e-12
        else:
            mix = (8192 / w - 1) / 3
            assert abs(f1 - ((1 - mix) * f0 / 8 + mix * f0)) < 1e-15


@pytest.mark.parametrize("kw", [dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, base=0.0),
                                dict(rotary_dim=8, scaling={"type": "other", "factor": 2}),
                                dict(rotary_dim=8, scaling={"type": "linear", "factor": 0}),
                                dict(rotary_dim=8, scaling={"type": "banded", "factor": 2, "original_max_positions": 8,
                                                            "low_freq_factor": 4, "high_freq_factor": 1})])
def test_bad_tables_are_refused(kw):
    with pytest.raises(ValueError):
        rotary_frequencies(**kw)


def test_cpu_tensors_are_refused():
    t = rotary_cos_sin(4, 8, device="cpu")
    x = torch.zeros(3, 2, 8, dtype=torch.float16)
    with pytest.raises(ValueError):
        apply_rotary_qk(x, x, t, torch.zeros(3, dtype=torch.int32))
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        append_rotary_paged_kv_cache(torch.zeros(1, 2, 2, 4, 8, dtype=torch.float16), None, x, x, i, i, i, i, t)


def test_c_entry_refuses_bad_arguments_without_a_gpu():
    import ctypes
    L = _lib.lib()
    a = _lib.RotaryArgs()
    a.num_tokens, a.num_qo_heads, a.head_dim, a.rotary_dim, a.max_positions = 4, 2, 64, 63, 10
    assert L.akt_rotary(ctypes.byref(a), None) == _lib.AKT_ERR_INVALID
    assert b"rotary_dim" in L.akt_last_error()
    a.rotary_dim = 128
    assert L.akt_rotary(ctypes.byref(a), None) == _lib.AKT_ERR_INVALID
    a.rotary_dim = 64
    assert L.akt_rotary(ctypes.byref(a), None) == _lib.AKT_ERR_INVALID  # no table
    a.num_tokens = 0
    assert L.akt_rotary(ctypes.byref(a), None) == _lib.AKT_OK
    x = _lib.AppendRotaryArgs()
    x.append.num_append, x.append.num_kv_heads, x.append.head_dim, x.append.page_size = 1, 0, 64, 16
    x.cos_sin, x.cos_sin_stride, x.rotary_dim = 16, 64, 64
    assert L.akt_append_rotary_paged_kv(ctypes.byref(x), None) == _lib.AKT_ERR_INVALID
    assert L.akt_rotary(None, None) == _lib.AKT_ERR_INVALID
    assert L.akt_append_rotary_paged_kv(None, None) == _lib.AKT_ERR_INVALID

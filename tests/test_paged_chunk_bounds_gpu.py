"""Chunk attention of a batch in which a sequence's query bounds are outside the rows."""
import math

import pytest
import torch

from attention_kernel_triton_b200 import _lib
from attention_kernel_triton_b200.paged_chunk_attention import chunk_paged_into, flash_attention_chunk_paged_with_lse
from test_paged_chunk_gpu import DEV, Case

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def device_status_clean():
    _lib.device_status(0, clear=True)
    yield


@pytest.mark.parametrize("B", [3, 120])
def test_rows_of_sequences_with_bad_query_bounds_are_zeros(B):
    c = Case([50] * B, [4] * B, Hkv=2, G=2, seed=2)
    T = 4 * B
    want, want_lse = flash_attention_chunk_paged_with_lse(*c.args())
    for at in ([4 * i for i in range(B)] + [T + 1],           # the last one's end is past the rows
               [-1] + [4 * i for i in range(1, B + 1)]):      # the first one's start is before them
        out = torch.full_like(c.q, math.nan)
        lse = torch.full(c.q.shape[:2], 5.0, device=DEV)
        chunk_paged_into(out, c.q, torch.tensor(at, dtype=torch.int32, device=DEV), *c.args()[2:], lse=lse)
        assert _lib.device_status(0, clear=True) == 4
        lost = slice(T - 4, T) if at[0] == 0 else slice(0, 4)
        keep = slice(0, T - 4) if at[0] == 0 else slice(4, T)
        assert (out[lost] == 0).all() and (lse[lost] == -math.inf).all()
        # (the work is cut differently, so the others are compared as values, outputs below 4)
        assert ((out[keep].float() - want[keep].float()).abs() <= 4 * 2.0 ** -9).all()
        assert ((lse[keep] - want_lse[keep]).abs() <= 1e-3).all()

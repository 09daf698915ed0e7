"""The evicting serving loop: shared prefix, weights, choice and eviction together, against dense attention."""
import importlib.util
import os

import pytest
import torch

from attention_kernel_triton_b200 import _lib

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("paged_eviction", os.path.join(ROOT, "examples", "paged_eviction.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_the_loop(example):
    _lib.device_status(0, clear=True)
    server = example.main(verbose=False)
    # fp16 rows, weights and outputs, a few roundings of 2^-11 on values below 4; the sums are fp32 of exponentials whose
    # exponents are off by less than 1e-5 (fp16 rows are exact, their products are summed in fp32)
    assert server.worst["attention"] <= 8e-3 and server.worst["sums"] <= 1e-4
    assert max(server.lens) <= server.budget + 12 and server.seen == [140] * 3
    assert _lib.device_status(0) == 0


@pytest.mark.parametrize("dtype,D,P", [(torch.bfloat16, 128, 16), (torch.float16, 64, 5), (torch.bfloat16, 64, 32)])
def test_pool_table_and_lists_stay_in_step(example, dtype, D, P):
    _lib.device_status(0, clear=True)
    s = example.EvictingServer(dtype=dtype, D=D, page_size=P, num_pages=400, budget=70, sinks=8, recent=20, seed=P)
    s.step(90)
    s.fork()
    for turn in range(4):
        for _ in range(3):
            s.step(1 + turn)
        keep, kept = s.evict()
        assert kept.tolist() == [70] * 3 and s.lens == [70] * 3
        # the lists have the format of the sparse decodes: ascending, the first and the last tokens among them
        assert (keep[..., 1:] > keep[..., :-1]).all() and same(keep[..., :8], torch.arange(8, device="cuda"))
        # every slot of the pool is the token that the lists say
        starts, indices, _ = s.table()
        for b in range(3):
            pages = indices[starts[b]:starts[b + 1]].long()
            rows = s.pool[pages].permute(1, 2, 0, 3, 4).flatten(2, 3)[:, :, :70].float()  # [2, Hkv, 70, D]
            assert same(rows, s.dense[b].permute(1, 2, 0, 3))
        assert (s.sums[:, :, 70:] == 0).all()
    assert _lib.device_status(0) == 0


def same(a, b):
    return bool((a == b).all())

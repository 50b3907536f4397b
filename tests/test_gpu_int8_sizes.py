"""Sizes past 32 bits (broadcast views, which take no memory) are refused, not cut to their low bits."""

from __future__ import annotations

import pytest
import torch

from pi05_fast.w4a4 import int8 as i8
from pi05_fast.w4a4 import kv_int8 as kv

pytestmark = pytest.mark.gpu
FAR = 1 << 32


def test_weight_rows(cuda):
    q = torch.ones((1, 16), dtype=torch.int8, device="cuda")
    with pytest.raises(RuntimeError, match="N must be at most"):
        i8.int8_gemm(q, torch.ones(1, device="cuda"), q.expand(FAR + 16, 16), torch.ones(1, device="cuda").expand(FAR + 16))


@pytest.mark.parametrize("b,t,pages", [(FAR + 1, 1, 1), (1, FAR + 1, 1), (1, 1, FAR + 1), (65536, 1, 1), (1, (1 << 24) + 1, 1)])
def test_cache_calls(cuda, b, t, pages):
    cache = kv.int8_kv_cache(2, 1, 64, "cuda")
    keep = [c.clone() for c in cache]
    k = torch.ones((1, 1, 1, 64), dtype=torch.float16, device="cuda").expand(b, t, 1, 64)
    table = torch.zeros((1, 1), dtype=torch.int32, device="cuda").expand(b, pages)
    lens = torch.zeros(1, dtype=torch.int32, device="cuda").expand(b)
    with pytest.raises(RuntimeError, match="at most"):
        kv.int8_kv_append(k, k, *cache, table, lens)
    assert all(torch.equal(a, c) for a, c in zip(keep, cache))
    with pytest.raises(RuntimeError, match="at most"):
        kv.int8_kv_attention(k, *cache, table, lens, 0.1)

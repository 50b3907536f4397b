"""Calls that write into an argument, on the direct route: autograd sees the change, as of torch's own calls."""

from __future__ import annotations

import pytest
import torch

from pi05_fast import w4a4

pytestmark = pytest.mark.gpu


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def test_adapters(cuda):
    y, x = (torch.randn((4, 64), device="cuda").half() for _ in range(2))
    a, b = torch.randn((1, 8, 64), device="cuda").half(), torch.randn((1, 64, 8), device="cuda").half()
    p = torch.ones_like(y, requires_grad=True)
    z = (y * p).sum()
    was = y._version
    w4a4.lora_add_(y[:, :], x, a, b, _i32([0] * 4))
    assert y._version > was
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()


def test_caches(cuda):
    k = torch.randn((2, 1, 1, 64), device="cuda").half()
    table, lens = _i32([[0], [1]]), _i32([0, 5])
    pos, freq = _i32([[0], [5]]), torch.ones(32, device="cuda")
    cache, cache8 = w4a4.kv_cache(2, 1, 64, torch.float16, "cuda"), w4a4.int8_kv_cache(2, 1, 64, "cuda")
    for call, written in ((lambda: w4a4.kv_append(k, k, *cache, table, lens), cache),
                          (lambda: w4a4.qk_norm_rope_append(k, k, k, None, None, 0.0, pos, freq, *cache, table, lens), cache),
                          (lambda: w4a4.int8_kv_append(k, k, *cache8, table, lens), cache8)):
        was = [t._version for t in written]
        call()
        assert all(t._version > v for t, v in zip(written, was))
    p = torch.ones_like(cache[1], requires_grad=True)
    z = (cache[1] * p).sum()
    w4a4.kv_append(k, k, *cache, table, lens)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()

"""The 8-bit operators under vmap: one call a sample, the same results."""

from __future__ import annotations

import pytest
import torch

from pi05_fast.w4a4 import int8 as i8
from pi05_fast.w4a4 import kv_int8 as kv

pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore:There is a performance drop")]


def test_vmap(cuda):
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((3, 5, 256), device="cuda", generator=gen).half()
    w, sw = i8.quantize_int8(torch.randn((40, 256), device="cuda", generator=gen).half())
    norm = torch.randn((256,), device="cuda", generator=gen).half()
    got = torch.vmap(lambda v: i8.add_rms_norm_int8(v, v, norm, 1e-6))(x)
    want = i8.add_rms_norm_int8(x, x, norm, 1e-6)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    y = torch.vmap(lambda q, s: i8.int8_gemm(q, s, w, sw))(want[0], want[1])
    assert torch.equal(y, i8.int8_gemm(want[0], want[1], w, sw))

    cache = kv.int8_kv_cache(4, 1, 64, "cuda")
    for c in cache[:2]:
        c.copy_(torch.randint(-127, 128, c.shape, device="cuda", generator=gen, dtype=torch.int8))
    for s in cache[2:]:
        s.fill_(0.01)
    q = torch.randn((3, 2, 4, 64), device="cuda", generator=gen).half()
    table, lens = torch.tensor([[0, 1], [2, 3], [1, 2]], dtype=torch.int32, device="cuda"), torch.tensor([70, 128, 3], dtype=torch.int32, device="cuda")
    got = torch.vmap(lambda a, b, n: kv.int8_kv_attention(a[None], *cache, b[None], n[None], 0.1)[0])(q, table, lens)
    assert torch.equal(got, kv.int8_kv_attention(q, *cache, table, lens, 0.1))

"""Chunks that cross the end of their table: a length past the table counts as the table's capacity, for the place of the
queries too, so that queries whose tokens were dropped are left out of ``q_lens`` and the others see what they should."""

from __future__ import annotations

import pytest
import torch
from test_gpu_kv_int8 import _gen, _i32, _kv, _pool

from pi05_fast.w4a4 import kv_int8 as kv

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("h,kvh,d,have,t", [(8, 1, 256, 190, 5), (4, 2, 128, 150, 200), (8, 2, 64, 60, 1100)])
def test_chunk_across_the_end(cuda, h, kvh, d, have, t):
    gen = _gen(d + t)
    pages = 3
    cache, table = _pool(gen, 1, pages + 20, kvh, d)
    short = table[:, :pages].contiguous()
    k, v = _kv(gen, 1, t, kvh, d, torch.float16)
    long_cache = [c.clone() for c in cache]
    kv.int8_kv_append(k, v, *cache, short, _i32([have]))
    kv.int8_kv_append(k, v, *long_cache, table, _i32([have]))
    kept = [c[short[0].long()] for c in cache]
    assert all(torch.equal(a, c[short[0].long()]) for a, c in zip(kept, long_cache))

    q = torch.randn((1, t, h, d), device="cuda", generator=gen).half()
    fit = pages * 64 - have
    # the queries that fit, as the last of a full table: those of a table that holds everything
    want = kv.int8_kv_attention(q[:, :fit], *long_cache, short, _i32([have + fit]), d**-0.5)
    got, lse = kv.int8_kv_attention(q, *cache, short, _i32([have + t]), d**-0.5, q_lens=_i32([fit]), return_lse=True)
    whole = kv.int8_kv_attention(q, *long_cache, table, _i32([have + t]), d**-0.5)
    torch.testing.assert_close(got[:, :fit], want, rtol=2e-3, atol=2e-3)
    torch.testing.assert_close(got[:, :fit], whole[:, :fit], rtol=2e-3, atol=2e-3)
    assert not got[:, fit:].any() and torch.isinf(lse[:, fit:]).all() and torch.isfinite(lse[:, :fit]).all()
    # past the table or at its end is the same
    assert torch.equal(got, kv.int8_kv_attention(q, *cache, short, _i32([pages * 64]), d**-0.5, q_lens=_i32([fit])))
    everything = kv.int8_kv_attention(q, *cache, short, _i32([10**9]), d**-0.5, causal=False)
    assert torch.equal(everything, kv.int8_kv_attention(q, *cache, short, _i32([pages * 64]), d**-0.5, causal=False))

"""Each form of the 16-bit KV attention (``kv_forms``) against 64 bits: lengths from one token to the table's, padding
queries, pages that no entry names, hidden junk, and values that only some queries see."""

from __future__ import annotations

import pytest
import torch
from kv_forms import FORMS
from test_gpu_kv import PAGE, TYPES, _check, _gen, _i32, _pool

from pi05_fast import w4a4

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kernel,waves,runs,shape", FORMS)
def test_against_64_bits(cuda, kernel, waves, runs, shape, dtype):
    b, t, h, kvh, d, pages = shape
    gen = _gen(sum(shape))
    cache, table = _pool(gen, b, pages, kvh, d, dtype)
    q = torch.randn((b, t, h, d), device="cuda", generator=gen).to(dtype)
    lens = torch.randint(1, pages * PAGE + 1, (b,), device="cuda", generator=gen).tolist()
    q_lens = torch.randint(1, t + 1, (b,), device="cuda", generator=gen).tolist()
    lens[0], lens[-1], q_lens[0] = pages * PAGE, min(t // 2 + 1, pages * PAGE), t
    if pages > 2:
        table[-1, 1] = -1
    dirty = [c.clone() for c in cache]
    for c in dirty:
        used = torch.zeros(c.size(0), PAGE, dtype=torch.bool, device="cuda")
        for i, n in enumerate(lens):
            for j in range((n + PAGE - 1) // PAGE):
                if table[i, j] >= 0:
                    used[table[i, j].long(), : min(n - PAGE * j, PAGE)] = True
        c.transpose(1, 2)[~used] = float("nan")
    for causal in (True, False):
        _check(q, dirty, table, lens, 0.07, causal, clean=cache)
    if t > 1:
        _check(q, dirty, table, lens, 0.07, True, q_lens, clean=cache)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kernel,waves,runs,shape", [f for f in FORMS if f[0] != "one"])
def test_values_that_some_queries_see(cuda, kernel, waves, runs, shape, dtype):
    """A NaN or infinity of the last tokens' values reaches the queries from its own on, in its dimension, and no others."""
    b, t, h, kvh, d, pages = shape
    gen = _gen(sum(shape) + 1)
    cache, table = _pool(gen, b, pages, kvh, d, dtype)
    q = torch.randn((b, t, h, d), device="cuda", generator=gen).to(dtype)
    n = pages * PAGE - 3
    lens = _i32([n] * b)
    want = w4a4.kv_attention(q, *cache, table, lens, 0.07)
    assert n >= t
    first = [t // 3, t - 1]  # key n - t + i is seen by queries i and later
    for bad in (float("nan"), float("inf")):
        dirty = cache[1].clone()
        hit = torch.zeros_like(want, dtype=torch.bool)
        for i, dim in zip(first, (5, d - 1)):
            key = n - t + i
            dirty[table[0, key // PAGE].long(), 0, key % PAGE, dim] = bad
            hit[0, i:, : h // kvh, dim] = True
        got = w4a4.kv_attention(q, cache[0], dirty, table, lens, 0.07)
        assert not torch.isfinite(got[hit]).any() and torch.equal(got[~hit], want[~hit])

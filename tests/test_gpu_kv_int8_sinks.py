"""Attention over the 8-bit cache where one key without a value takes nearly all of a row's mass.

All keys but one score zero, so that they share one weight w = 1 / (e^z + n - 1), z the score of the one; its values
are zero and the others' positive, so that the output is w times their sum and nothing cancels.

Tolerance, relative.  The one key's weight is held between 2^7 and 2^15, so the others' are at least 2^7 e^-z, and a
rounding to fp16 is within half a step of the normal range, 2^-11, or below it 2^-25 / (2^7 e^-z).  Queries
are held to 1 / 65024 of their maximum, so z is within z / 65024, which moves w by as much; fp32 roundings and the
exponential of z and the scale's logarithm 2^-19 (z + 8), the accumulation 2^-18, the output half a step.
"""

from __future__ import annotations

import pytest
import torch

from pi05_fast.w4a4 import kv_int8 as kv

pytestmark = pytest.mark.gpu


def _sinks(b, t, h, kvh, d, n, dtype, seed):
    """Cache, table, queries and the exact rows' (z, out): the first key of each sequence is the sink."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    pages = (n + 63) // 64
    cache = kv.int8_kv_cache(b * pages, kvh, d, "cuda")
    table = torch.randperm(b * pages, device="cuda", generator=gen).to(torch.int32).view(b, pages)
    cache[0][table[:, 0].long(), :, 0, 0] = 127
    cache[1].copy_(torch.randint(1, 128, cache[1].shape, device="cuda", generator=gen, dtype=torch.int8))
    cache[1][table[:, 0].long(), :, :, 0] = 0
    cache[2].fill_(0.02)
    cache[3].fill_(0.03)
    q = torch.randn((b, t, h, d), device="cuda", generator=gen)
    q[..., 0] = 4 + 6 * torch.rand((b, t, h), device="cuda", generator=gen)
    q[..., 1:].clamp_(-4, 4)
    q = q.to(dtype)
    scaling = 17 / (10 * 127 * float(cache[2][0, 0]))  # z from 6.8 to 17: sinks of 0.1 to 0.999 and above
    z = q[..., 0].double() * 127 * cache[2][0, 0].double() * scaling
    v = cache[1].double() * cache[3][0, 0].double()
    total = torch.stack([torch.cat([v[i] for i in row.tolist()], -1)[..., :n].sum(-1) for row in table])  # [B, KVH, D]
    w = 1 / (torch.exp(z) + n - 1)
    out = w[..., None] * total.repeat_interleave(h // kvh, 1)[:, None]
    return cache, table, q, scaling, z, out


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("b,t,h,kvh,d,n", [
    (1, 1, 8, 1, 256, 8192), (64, 1, 8, 1, 256, 8000), (1, 1, 8, 8, 64, 8192), (8, 50, 8, 1, 256, 826), (2, 776, 8, 1, 256, 4096),
    (2, 776, 8, 2, 128, 8192), (4, 1501, 8, 2, 64, 8000), (1, 16, 1, 1, 128, 32768), (2, 3000, 8, 1, 256, 8192),
])
def test_small_weights_beside_a_sink(cuda, b, t, h, kvh, d, n, dtype):
    cache, table, q, scaling, z, out = _sinks(b, t, h, kvh, d, n, dtype, t + n + d)
    lens = torch.full((b,), n, dtype=torch.int32, device="cuda")
    got, lse = kv.int8_kv_attention(q, *cache, table, lens, scaling, causal=False, return_lse=True)
    small = torch.maximum(torch.full_like(z, 2.0**-11), 2.0**-32 * torch.exp(z))
    rel = small + 2 * z / 65024 + 2.0**-19 * (z + 8) + 2.0**-18
    tol = rel[..., None] * out + torch.finfo(dtype).eps / 2 * 1.001 * out + 2.0**-25
    assert ((got.double() - out).abs() / tol).max().item() <= 1
    want = torch.log(torch.exp(z) + n - 1)
    assert ((lse.double() - want).abs() <= z / 65024 + 2.0**-19 * (z + 8) + 2e-7 * want).all()

"""How many bits of an fp32 weight the 16-bit serving operators' second products keep, seen where large terms cancel.

Attention.  Of three keys the second cancels the first and the third what its rounding left, so that the output is
below 2^-14 of the terms and its own rounding does not hide theirs.  A logit is one product, exact, of at
most 1.  In units of 2^-24: the exponent s = log2(e) z is 0.4 off by the constant and 1 by its rounding, less the
reference (at most 7 in size) 4, together 5.4 ln 2 = 3.8 of the weight; exp2 2; two parts of fp16 4, three of bf16
nothing; two additions of three products, truncated at worst, 4.  The sum of the weights scales the small output
only.

Adapters.  The two ranks of a row are whole numbers of up to 24 bits (fp16: 22), made by two products, and all but
cancel: every sum is exact in fp32, so that the result is compared bit for bit.
"""

from __future__ import annotations

import pytest
import torch

from pi05_fast import w4a4

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def cancelling(gen, b, d, dtype, device="cuda"):
    """z [B, 3], v [B, 3, D] in the type, the weighted sum of v and the size of its terms."""
    z = (torch.rand((b, 3), device=device, generator=gen) * 2 - 1).to(dtype).double()
    p = torch.softmax(z, -1)[..., None]
    v = torch.zeros((b, 3, d), dtype=torch.float64, device=device)
    v[:, 0] = (torch.randn((b, d), device=device, generator=gen) * 64).to(dtype).double()
    v[:, 1] = (-p[:, 0] * v[:, 0] / p[:, 1]).to(dtype).double()
    v[:, 2] = (-(p[:, :2] * v[:, :2]).sum(1) / p[:, 2]).to(dtype).double()
    return z, v, (p * v).sum(1), (p * v.abs()).sum(1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,t,h,kvh,d", [(200, 1, 1, 1, 256), (200, 1, 4, 1, 128), (200, 1, 2, 2, 64), (60, 3, 1, 1, 256), (60, 5, 2, 1, 128),
                                         (60, 9, 1, 1, 64), (70, 64, 8, 1, 256), (70, 70, 8, 1, 128), (70, 90, 8, 1, 64)])
def test_attention_weights(cuda, b, t, h, kvh, d, dtype):
    gen = _gen(b + t + d)
    z, v, want, size = cancelling(gen, b, d, dtype)
    cache = w4a4.kv_cache(b, kvh, d, dtype, "cuda")
    cache[0][:, :, :3, 0] = z.to(dtype)[:, None]
    cache[1][:, :, :3] = v.to(dtype)[:, None]
    q = torch.zeros((b, t, h, d), dtype=dtype, device="cuda")
    q[..., 0] = 1
    table = torch.arange(b, device="cuda", dtype=torch.int32)[:, None]
    lens = torch.full((b,), 3, dtype=torch.int32, device="cuda")
    got = w4a4.kv_attention(q, *cache, table, lens, 1.0, causal=False).double()
    units = 10.0 if dtype == torch.bfloat16 else 14.0
    tol = units * 2.0**-24 * size + torch.finfo(dtype).eps / 2 * 1.001 * want.abs() + 2.0**-25
    over = ((got - want[:, None, None]).abs() / tol[:, None, None]).max().item()
    assert over <= 1, over


def _far_sums(gen, m, k, dtype):
    """x [M, K] and, for one adapter a row, the first factors of two ranks [M, K] with whole sums of up to 24 (fp16: 22) bits
    that are less than 100 apart; the sums."""
    bits, parts = (8, 3) if dtype == torch.bfloat16 else (11, 2)
    top = 1 << (bits * parts)
    h0 = torch.randint(top // 2, top - 200, (m,), device="cuda", generator=gen)
    h1 = h0 + torch.randint(-100, 101, (m,), device="cuda", generator=gen)
    at = torch.randperm(k, device="cuda", generator=gen)[:parts]
    x = torch.zeros((m, k), device="cuda")
    a = torch.zeros((m, 2, k), device="cuda")
    for i in range(parts):
        x[:, at[i]] = float(1 << (bits * i))
        for j, h in enumerate((h0, h1)):
            a[:, j, at[i]] = ((h >> (bits * i)) & ((1 << bits) - 1)).float()
    return x.to(dtype), a.to(dtype), h0 - h1


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("per_id", [1, 5, 70])
@pytest.mark.parametrize("r,k,n", [(8, 64, 40), (24, 104, 130), (64, 128, 300), (128, 64, 96), (8, 16384, 64), (24, 4096, 257), (64, 2048, 130),
                                   (128, 2048, 70)])
def test_sums_of_adapters(cuda, r, k, n, per_id, dtype):
    """In one launch (the first four) and in two."""
    gen = _gen(r + k + n + per_id)
    count = 9
    x, two, apart = _far_sums(gen, count, k, dtype)
    a = torch.zeros((count, r, k), dtype=dtype, device="cuda")
    b = torch.zeros((count, n, r), dtype=dtype, device="cuda")
    i, j = (0, r - 1) if per_id == 1 else (r // 2, r // 2 + 1)
    a[:, i], a[:, j], b[:, :, i], b[:, :, j] = two[:, 0], two[:, 1], 1, -1
    ids = torch.randperm(count, device="cuda", generator=gen)
    rows = ids.repeat_interleave(per_id)
    y = torch.randint(-100, 101, (count * per_id, n), device="cuda", generator=gen).to(dtype)
    want = (y.float() + apart[rows, None]).to(dtype)
    got = w4a4.lora_add(y.view(count, per_id, n), x[rows].view(count, per_id, k), a, b, ids.to(torch.int32))
    assert torch.equal(got.view(-1, n), want)


@pytest.mark.parametrize("b,t,h,kvh,d,pages", [(3, 1, 8, 1, 256, 3), (2, 1, 4, 1, 128, 40), (40, 1, 4, 2, 64, 2), (3, 9, 4, 1, 256, 3),
                                               (3, 20, 2, 1, 64, 4), (6, 110, 8, 1, 256, 5), (12, 97, 8, 2, 128, 5), (70, 70, 3, 1, 64, 5)])
def test_values_at_the_end_of_the_range(cuda, b, t, h, kvh, d, pages):
    """bf16 values of nearly fp32's largest number, of one sign and of both: their mean is as large at most."""
    from test_gpu_kv import _check, _pool

    gen = _gen(b + t + d)
    cache, table = _pool(gen, b, pages, kvh, d, torch.bfloat16)
    q = (torch.randn((b, t, h, d), device="cuda", generator=gen) * 3).bfloat16()
    lens = torch.randint(1, pages * 64 + 1, (b,), device="cuda", generator=gen).tolist()
    lens[0] = pages * 64
    for v in (torch.full_like(cache[1], torch.finfo(torch.bfloat16).max), (torch.rand(cache[1].shape, device="cuda", generator=gen) * 3.3e38).bfloat16(),
              cache[1].sign() * 3e38):
        _check(q, [cache[0], v.bfloat16()], table, lens, d**-0.5, causal=False)
        _check(q, [cache[0], v.bfloat16()], table, lens, d**-0.5)

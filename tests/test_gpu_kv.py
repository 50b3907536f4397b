"""Attention over the 16-bit KV cache against 64 bits.

Tolerance.  A logit is |scaling| D 2^-23 (|q| |k|^T) off (D products, exact in fp32, summed in any order and
truncated at worst) and 2^-21 of its size (the product with the scale, the difference in the exponent and
exp2): e in all.  A probability is then 2 e off relatively.  Its two 16-bit parts hold it to 2^-18 (bf16), or
2^-22 and 2^-32 of the row's largest weight (fp16); sums of n terms, once for the weights and twice for their products
with V, 3 n 2^-23.  The output is half a step of its type.
"""

from __future__ import annotations

import pytest
import torch

from pi05_fast import w4a4

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16]
PAGE = 64


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _pool(gen, b, table_pages, kvh, d, dtype, spare=2):
    n = b * table_pages + spare
    cache = [torch.randn((n, kvh, PAGE, d), device="cuda", generator=gen).to(dtype) for _ in range(2)]
    table = torch.randperm(n, device="cuda", generator=gen)[: b * table_pages].to(torch.int32).view(b, table_pages)
    return cache, table


def _reference(q, cache, table, lens, scaling, causal, q_lens):
    """out, lse and bounds (float64).  What is hidden is taken as zeros."""
    kc, vc = cache
    b, t, h, d = q.shape
    kvh = kc.size(1)
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    lse = torch.full((b, t, h), float("-inf"), dtype=torch.float64, device="cuda")
    ltol = torch.zeros_like(lse)
    part = 2.0**-18 if q.dtype == torch.bfloat16 else 2.0**-22
    for i in range(b):
        n, ql = min(max(lens[i], 0), table.size(1) * PAGE), t if q_lens is None else min(max(q_lens[i], 0), t)
        if n == 0 or ql == 0:
            continue
        ids = table[i].long()
        ok = ((ids >= 0) & (ids < kc.size(0))).repeat_interleave(PAGE)[:n]
        ids = ids.clamp(0, kc.size(0) - 1)
        at = torch.arange(n, device="cuda")
        last = n - ql + torch.arange(ql, device="cuda") if causal else torch.full((ql,), n, device="cuda")
        see = ok & (at <= last[:, None])
        for g in range(kvh):
            k, v = (torch.where(ok[:, None], c[ids, g].double().reshape(-1, d)[:n], 0.0) for c in (kc, vc))
            for hh in range(g * (h // kvh), (g + 1) * (h // kvh)):
                qq = q[i, :ql, hh].double()
                z = (qq @ k.t().contiguous() * scaling).masked_fill(~see, float("-inf"))
                p = torch.softmax(z, -1).nan_to_num(0)
                size = (qq.abs() @ k.abs().t().contiguous() * abs(scaling)).masked_fill(~see, 0.0).amax(-1, keepdim=True)
                e = size * (d * 2.0**-23 + 2.0**-21)
                out[i, :ql, hh] = p @ v
                lse[i, :ql, hh] = torch.logsumexp(z, -1)
                tol[i, :ql, hh] = (2 * e + part + 3 * n * 2.0**-23) * (p @ v.abs()) * 1.01 + n * 2.0**-32 * v.abs().max()
                ltol[i, :ql, hh] = (e + n * 2.0**-23 + 2.0**-20)[:, 0] + 2.0**-21 * lse[i, :ql, hh].abs()
    some = torch.isfinite(lse)[..., None]
    tol = torch.where(some, tol + torch.finfo(q.dtype).eps / 2 * 1.001 * out.abs() + 2.0**-25, 0.0)
    return out, lse, tol, ltol


def _check(q, cache, table, lens, scaling, causal=True, q_lens=None, clean=None):
    """clean: the cache with zeros in the place of what may hold anything."""
    got, lse = w4a4.kv_attention(q, *cache, table, _i32(lens), scaling, causal=causal, q_lens=None if q_lens is None else _i32(q_lens),
                                 return_lse=True)
    q0 = torch.where(torch.isfinite(q), q, torch.zeros_like(q))
    want, wlse, tol, ltol = _reference(q0, cache if clean is None else clean, table, lens, scaling, causal, q_lens)
    assert torch.isfinite(got).all() and got.dtype == q.dtype
    over = (got.double() - want).abs() - tol
    assert (over <= 0).all(), over.max().item()
    none = torch.isinf(wlse)
    assert torch.equal(none, torch.isinf(lse)) and not got[none].any()
    assert ((lse.double() - wlse).abs() <= ltol)[~none].all()
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("h,kvh,d", [(8, 1, 256), (6, 2, 128), (5, 5, 64), (40, 2, 64), (1, 1, 256), (32, 8, 128)])
@pytest.mark.parametrize("lens,t", [([1], 1), ([0, 64, 65], 1), ([31, 32, 33, 63], 1), ([63, 300, 1000, 7], 1), ([130, 5, 64], 5),
                                    ([70, 200], 50)])
def test_attention(cuda, lens, t, h, kvh, d, dtype):
    gen = _gen(t + h + d)
    b = len(lens)
    cache, table = _pool(gen, b, (max(lens) + 63) // 64 + 1, kvh, d, dtype)
    q = (torch.randn((b, t, h, d), device="cuda", generator=gen) * 1.5).to(dtype)
    for causal in (True, False):
        _check(q, cache, table, lens, d**-0.5, causal)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("h,kvh,d,b,pages", [(8, 1, 256, 1, 130), (8, 1, 256, 70, 20), (32, 8, 128, 3, 64), (8, 8, 64, 40, 17), (8, 1, 256, 2, 13),
                                             (4, 2, 128, 300, 3)])
def test_decode(cuda, h, kvh, d, b, pages, dtype):
    """One token a sequence over lengths from one token to the table's, in runs and without."""
    gen = _gen(b + pages)
    cache, table = _pool(gen, b, pages, kvh, d, dtype)
    q = (torch.randn((b, 1, h, d), device="cuda", generator=gen) * 1.5).to(dtype)
    lens = torch.randint(1, pages * PAGE + 1, (b,), device="cuda", generator=gen).tolist()
    lens[0] = pages * PAGE
    if b > 2:
        lens[1], lens[2] = 1, 0
    _check(q, cache, table, lens, d**-0.5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("h,kvh,d", [(8, 1, 256), (4, 4, 128), (10, 2, 64)])
def test_ragged_queries(cuda, h, kvh, d, dtype):
    """Padding queries, sequences shorter than their queries, and none at all: zeros."""
    gen = _gen(11)
    cache, table = _pool(gen, 5, 5, kvh, d, dtype)
    q = torch.randn((5, 40, h, d), device="cuda", generator=gen).to(dtype)
    q[2] = float("nan")  # a sequence without queries
    q[3, 7:] = float("inf")  # behind the last query
    for causal in (True, False):
        _check(q, cache, table, [300, 10, 64, 200, 0], 0.06, causal, [40, 25, 0, 7, 33])
        _check(q[:, :1].contiguous(), cache, table, [300, 10, 64, 200, 0], 0.06, causal, [1, 1, 0, 1, -3])


def test_table_edges(cuda):
    """Lengths past the table, entries that name no page, sequences that share pages, no pages at all."""
    gen = _gen(12)
    cache, table = _pool(gen, 4, 3, 1, 128, torch.float16)
    table[1] = table[0]
    table[2, 1] = -1
    table[3, 0] = 10**9
    for t in (1, 2, 20):
        q = torch.randn((4, t, 4, 128), device="cuda", generator=gen).half()
        _check(q, cache, table, [192, 100, 192, 150], 0.09)
        _check(q, cache, table, [10**6, -3, 70, 30], 0.09, causal=False)
        wide = torch.full((4, 9), -1, dtype=torch.int32, device="cuda")
        wide[:, 2:5] = table
        a = w4a4.kv_attention(q, *cache, wide[:, 2:5], _i32([192, 100, 50, 150]), 0.09)
        assert torch.equal(a, w4a4.kv_attention(q, *cache, table, _i32([192, 100, 50, 150]), 0.09))
    assert not w4a4.kv_attention(q, *w4a4.kv_cache(0, 1, 128, torch.float16, "cuda"), table, _i32([5] * 4), 0.1).any()
    assert not w4a4.kv_attention(q, *cache, table[:, :0], _i32([5] * 4), 0.1).any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("junk", [float("nan"), float("inf"), -float("inf"), 60000.0])
def test_hidden_junk(cuda, junk, dtype):
    """What no query sees has no effect, whatever it holds: rows behind the last token, pages not reached, pages
    that an entry of the table does not name."""
    gen = _gen(13)
    for h, kvh, d in ((8, 1, 256), (4, 2, 64)):
        cache, table = _pool(gen, 3, 4, kvh, d, dtype)
        table[2, 0] = -1
        lens = [100, 129, 200]
        dirty = [c.clone() for c in cache]
        for c in dirty:
            used = torch.zeros(c.size(0), PAGE, dtype=torch.bool, device="cuda")
            for i, n in enumerate(lens):
                for p in range((n + 63) // 64):
                    if table[i, p] >= 0:
                        used[table[i, p].long(), : min(n - 64 * p, 64)] = True
            c.transpose(1, 2)[~used] = junk
        for t in (1, 30):
            q = torch.randn((3, t, h, d), device="cuda", generator=gen).to(dtype)
            for causal in (True, False):
                want = _check(q, cache, table, lens, 0.06, causal)
                got = w4a4.kv_attention(q, *dirty, table, _i32(lens), 0.06, causal=causal)
                assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("h,kvh,d,b,t", [(8, 1, 256, 6, 110), (8, 2, 128, 12, 97), (3, 1, 64, 70, 70), (40, 2, 64, 5, 83)])
def test_many_rows(cuda, h, kvh, d, b, t, dtype):
    """More than one round of 16 rows a workgroup: tiles of tokens across each other, lengths below the queries', padding
    queries, pages that no entry names, hidden junk."""
    gen = _gen(b + t)
    cache, table = _pool(gen, b, 5, kvh, d, dtype)
    table[1, 1], table[2, 0] = -1, cache[0].size(0)
    q = torch.randn((b, t, h, d), device="cuda", generator=gen).to(dtype)
    lens = torch.randint(1, 5 * PAGE + 1, (b,), device="cuda", generator=gen).tolist()
    lens[:5] = [300, 130, 190, 64, 33]
    q_lens = torch.randint(0, t + 1, (b,), device="cuda", generator=gen).tolist()
    q_lens[:3] = [t, t - 1, 40]
    dirty = [c.clone() for c in cache]
    for c in dirty:
        used = torch.zeros(c.size(0), PAGE, dtype=torch.bool, device="cuda")
        for i, n in enumerate(lens):
            for j in range((n + 63) // 64):
                if 0 <= table[i, j] < c.size(0):
                    used[table[i, j].long(), : min(n - 64 * j, 64)] = True
        c.transpose(1, 2)[~used] = float("nan")
    for causal in (True, False):
        _check(q, dirty, table, lens, 0.07, causal, clean=cache)
        _check(q, dirty, table, lens, 0.07, causal, q_lens, clean=cache)


@pytest.mark.parametrize("dtype", TYPES)
def test_nonfinite_values_of_many_rows(cuda, dtype):
    gen = _gen(15)
    for h, kvh, d in ((8, 1, 256), (8, 2, 128), (3, 1, 64)):
        b, t = 1200 * 16 // (100 * h // kvh) // kvh, 100
        cache, table = _pool(gen, b, 4, kvh, d, dtype)
        q = torch.randn((b, t, h, d), device="cuda", generator=gen).to(dtype)
        lens = _i32([200] * b)
        want = w4a4.kv_attention(q, *cache, table, lens, 0.06)
        for bad in (float("nan"), float("inf")):
            dirty = cache[1].clone()
            # keys 110 and 180 are seen by queries 10 and later, 80 and later (100 + i >= key)
            dirty[table[0, 1].long(), 0, 110 - 64, 5] = bad
            dirty[table[0, 2].long(), 0, 180 - 128, d - 1] = bad
            got = w4a4.kv_attention(q, cache[0], dirty, table, lens, 0.06)
            hit = torch.zeros_like(got, dtype=torch.bool)
            hit[0, 10:, : h // kvh, 5] = hit[0, 80:, : h // kvh, d - 1] = True
            assert not torch.isfinite(got[hit]).any() and torch.equal(got[~hit], want[~hit])


@pytest.mark.parametrize("dtype", TYPES)
def test_nonfinite_values_reach_only_who_sees_them(cuda, dtype):
    gen = _gen(14)
    for h, kvh, d in ((8, 1, 256), (4, 2, 128), (2, 2, 64)):
        cache, table = _pool(gen, 1, 4, kvh, d, dtype)
        q = torch.randn((1, 40, h, d), device="cuda", generator=gen).to(dtype)
        lens = _i32([200])
        want = w4a4.kv_attention(q, *cache, table, lens, 0.06)
        for side in (0, 1):
            for bad in (float("nan"), float("inf")):
                dirty = [c.clone() for c in cache]
                # key 180 is seen by queries 20 and later (160 + i >= 180)
                dirty[side][table[0, 2].long(), 0, 180 - 128, 5] = bad
                got = w4a4.kv_attention(q, *dirty, table, lens, 0.06)
                assert torch.equal(got[:, :20], want[:, :20])
                group = h // kvh
                assert torch.equal(got[:, :, group:], want[:, :, group:])
                if side == 1:
                    assert torch.isnan(got[:, 20:, :group, 5]).all() if bad != bad else not torch.isfinite(got[:, 20:, :group, 5]).any()
                    rest = [j for j in range(d) if j != 5]
                    assert torch.equal(got[..., rest], want[..., rest])
                elif bad != bad:
                    assert torch.isnan(got[:, 20:, :group]).all()


def test_extremes(cuda):
    """Flat and peaked rows, scores far from zero, a query that is not finite."""
    gen = _gen(15)
    for dtype in TYPES:
        cache, table = _pool(gen, 2, 10, 1, 256, dtype)
        q = torch.randn((2, 3, 8, 256), device="cuda", generator=gen).to(dtype)
        for scaling in (0.0, 0.0625, 1.0, 8.0, -0.0625):
            _check(q, cache, table, [640, 600], scaling)
        _check(q * 0, cache, table, [640, 600], 0.0625)
        _check((q * 3000).clamp(-60000, 60000), cache, table, [640, 600], 1e-5)
        # all scores of a row far below zero
        low = [cache[0].abs() * 20, cache[1]]
        _check(-q.abs() * 20, low, table, [640, 600], 1.0)
        bad = q.clone()
        bad[1, 2, 3, 100] = float("nan")
        got = w4a4.kv_attention(bad, *cache, table, _i32([640, 600]), 0.0625)
        assert torch.isnan(got[1, 2, 3]).all()
        got[1, 2, 3] = 0
        assert torch.isfinite(got).all()
    b = torch.randn((2, 1, 8, 256), device="cuda", generator=gen).bfloat16()
    _check(b * 1e30, cache, table, [640, 600], 6e-32)
    _check(b * 1e-30, cache, table, [640, 600], 6e28)


@pytest.mark.parametrize("dtype", TYPES)
def test_many_small_weights_beside_a_large_one(cuda, dtype):
    """A key without a value takes nearly all of the mass; thousands of others share the rest."""
    gen = _gen(16)
    cache, table = _pool(gen, 2, 100, 1, 128, dtype)
    cache[0].zero_()
    cache[1].copy_(torch.rand(cache[1].shape, device="cuda", generator=gen) + 0.5)
    q = torch.zeros((2, 1, 4, 128), device="cuda", dtype=dtype)
    q[..., 0] = 4
    for where in (0, 6399, 3210):
        for gap in (6.0, 12.0, 16.0):
            page = table[:, where // 64].long()
            c = [x.clone() for x in cache]
            c[0][page, 0, where % 64, 0] = gap / 4
            c[1][page, 0, where % 64] = 0
            got, lse = w4a4.kv_attention(q, *c, table, _i32([6400, 6400]), 1.0, return_lse=True)
            z = torch.zeros(6400, dtype=torch.float64, device="cuda")
            z[where] = float(torch.tensor(gap / 4).to(dtype)) * 4
            p = torch.softmax(z, 0)
            for i in range(2):
                v = c[1][table[i].long(), 0].double().reshape(-1, 128)
                want = p @ v
                # n 2^-32 of the largest weight beside the terms' own relative errors, 3 n 2^-23 at worst
                tol = want.abs() * (2.0**-17 + 3 * 6400 * 2.0**-23 + torch.finfo(dtype).eps / 2 * 1.001) + p.max() * 6400 * 2.0**-32 * 1.5 + 2.0**-25
                assert ((got[i, 0].double() - want).abs() <= tol).all()


def test_long(cuda):
    gen = _gen(17)
    for dtype in TYPES:
        cache, table = _pool(gen, 2, 520, 1, 256, dtype)
        q = torch.randn((2, 1, 8, 256), device="cuda", generator=gen).to(dtype)
        _check(q, cache, table, [33000, 1], 0.0625)
        _check(q, cache, table, [33280, 20000], 0.0, causal=False)
    q = torch.randn((2, 300, 8, 256), device="cuda", generator=gen).to(dtype)
    _check(q, cache, table, [5000, 333], 0.0625)


def test_pool_past_4_gib(cuda):
    gen = _gen(18)
    small, _ = _pool(gen, 1, 4, 1, 256, torch.bfloat16, spare=0)
    n = 140000
    big = w4a4.kv_cache(n, 1, 256, torch.bfloat16, "cuda")
    ids = torch.tensor([n - 1, 135000, 5, n - 2], device="cuda")
    for c, part in zip(big, small):
        c[ids] = part
    q = torch.randn((1, 2, 8, 256), device="cuda", generator=gen).bfloat16()
    a = w4a4.kv_attention(q, *big, ids.to(torch.int32).view(1, 4), _i32([250]), 0.06)
    assert torch.equal(a, w4a4.kv_attention(q, *small, _i32([[0, 1, 2, 3]]), _i32([250]), 0.06))


def test_query_strides(cuda):
    gen = _gen(19)
    cache, table = _pool(gen, 3, 4, 1, 256, torch.float16)
    wide = torch.randn((3, 6, 2560), device="cuda", generator=gen).half()
    q = wide[:, :, :2048].view(3, 6, 8, 256)
    lens = _i32([200, 65, 6])
    want = w4a4.kv_attention(q.contiguous(), *cache, table, lens, 0.06)
    assert torch.equal(w4a4.kv_attention(q, *cache, table, lens, 0.06), want)
    turned = q.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(w4a4.kv_attention(turned, *cache, table, lens, 0.06), want)
    odd = torch.zeros((3, 6, 8, 257), device="cuda", dtype=torch.float16)
    odd[..., 1:] = q
    assert torch.equal(w4a4.kv_attention(odd[..., 1:], *cache, table, lens, 0.06), want)
    one = q[:, :1, :1].expand(3, 6, 8, 256)
    assert torch.equal(w4a4.kv_attention(one, *cache, table, lens, 0.06), w4a4.kv_attention(one.contiguous(), *cache, table, lens, 0.06))


def test_joined_with_other_keys(cuda):
    """Two halves of a cache joined by their lse are the whole."""
    gen = _gen(20)
    cache, table = _pool(gen, 2, 6, 1, 256, torch.float16)
    q = torch.randn((2, 4, 8, 256), device="cuda", generator=gen).half()
    parts = [w4a4.kv_attention(q, *cache, tb, _i32(n), 0.06, causal=False, return_lse=True)
             for tb, n in ((table[:, :3], [192, 192]), (table[:, 3:], [180, 20]))]
    whole, lse = w4a4.kv_attention(q, *cache, table, _i32([372, 212]), 0.06, causal=False, return_lse=True)
    both = torch.logaddexp(parts[0][1], parts[1][1])
    joined = sum(o.float() * torch.exp(ls - both)[..., None] for o, ls in parts)
    assert (both - lse).abs().max() < 1e-4
    # three roundings to fp16 of values of at most 1
    assert (joined - whole.float()).abs().max() < 3 * 2.0**-11


# ------------------------------------------------------------------ the operators together
class Layer:
    """The attention half of a layer for a batch of requests with adapters."""

    def __init__(self, gen, width, h, kvh, d, dtype):
        def rand(*s, scale=1.0):
            return (torch.randn(s, device="cuda", generator=gen) * scale).to(dtype)

        self.h, self.kvh, self.d, self.dtype = h, kvh, d, dtype
        self.norm = rand(width, scale=0.1)
        self.qkv = w4a4.quantize_int8(rand((h + 2 * kvh) * d, width, scale=0.05))
        self.o = w4a4.quantize_int8(rand(width, h * d, scale=0.05))
        self.widths = [h * d, kvh * d, kvh * d]
        self.qkv_a, self.qkv_b = rand(3, 3 * 8, width, scale=width**-0.5), rand(3, (h + 2 * kvh) * d, 8, scale=0.3)
        self.o_a, self.o_b = rand(3, 16, h * d, scale=(h * d)**-0.5), rand(3, width, 16, scale=0.3)
        self.scale = torch.tensor([1.0, 0.5, 2.0], device="cuda")
        self.qw, self.kw = rand(d, scale=0.2), rand(d, scale=0.2)
        self.freq = (10000.0 ** (-torch.arange(d // 2, device="cuda", dtype=torch.float64) / (d // 2))).float()

    def __call__(self, x, res, ids, pos, cache, table, lens, keep=None):
        b, t, _ = x.shape
        h, kvh, d = self.h, self.kvh, self.d
        q8, s, hid = w4a4.add_rms_norm_int8(x, res, self.norm, 1e-6)
        base = w4a4.int8_gemm(q8, s, *self.qkv, out_dtype=self.dtype)
        qkv = w4a4.lora_add(base, hid, self.qkv_a, self.qkv_b, ids, self.scale, slices=self.widths)
        heads = qkv.view(b, t, h + 2 * kvh, d)
        k, v = heads[:, :, h:h + kvh], heads[:, :, h + kvh:]
        q = w4a4.qk_norm_rope_append(heads[:, :, :h], k, v, self.qw, self.kw, 1e-6, pos, self.freq, *cache, table, lens)
        att = w4a4.kv_attention(q, *cache, table, lens + t, d**-0.5)
        a8, sa = w4a4.quantize_int8(att.view(b, t, -1))
        y = w4a4.int8_gemm(a8, sa, *self.o, residual=hid, out_dtype=self.dtype)
        w4a4.lora_add_(y, att.view(b, t, -1), self.o_a, self.o_b, ids, self.scale)
        if keep is not None:
            keep.update(base=base, hid=hid, qkv=qkv, k=k, v=v, q=q, att=att)
        return y


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_half_of_a_layer(cuda, dtype):
    """A prompt in two chunks and then single tokens, three requests, two of them with an adapter: the cache holds what the
    separate calls give, and the attention of each step is that of its inputs in 64 bits."""
    gen = _gen(21)
    layer = Layer(gen, 512, 4, 1, 128, dtype)
    b, ids = 3, _i32([2, -1, 0])
    cache, table = _pool(gen, b, 4, 1, 128, dtype)
    have = 0
    for t in (90, 37, 1, 1, 1):
        x, res = (torch.randn((b, t, 512), device="cuda", generator=gen).to(dtype) for _ in range(2))
        pos = (have + torch.arange(t, device="cuda"))[None].expand(b, t)
        lens, was, got = _i32([have] * b), [c.clone() for c in cache], {}
        layer(x, res, ids, pos, cache, table, lens, keep=got)
        # the parts of the joined projection one by one
        at = 0
        for g, width in enumerate(layer.widths):
            part = got["base"][..., at:at + width]
            one = w4a4.lora_add(part, got["hid"], layer.qkv_a[:, 8 * g:8 * g + 8], layer.qkv_b[:, at:at + width], ids, layer.scale)
            # the same sums in another order: fp32, and one rounding
            step = torch.finfo(dtype).eps * one.float().abs() + 2.0**-12 * part.float().abs().amax()
            assert ((got["qkv"][..., at:at + width].float() - one.float()).abs() <= step).all()
            at += width
        assert torch.equal(got["qkv"][1], got["base"][1])
        heads = got["qkv"].view(b, t, 6, 128)
        q, k = w4a4.qk_norm_rope(heads[:, :, :4], heads[:, :, 4:5], layer.qw, layer.kw, 1e-6, pos, layer.freq)
        w4a4.kv_append(k, got["v"], *was, table, lens)
        assert torch.equal(q, got["q"]) and all(torch.equal(a, c) for a, c in zip(was, cache))
        have += t
        want, _, tol, _ = _reference(q, cache, table, [have] * b, 128**-0.5, True, None)
        assert ((got["att"].double() - want).abs() <= tol).all()


def test_captured_decode_steps(cuda):
    """A captured step, replayed with moving lengths and adapters, does what the eager steps do; two graphs on their own
    caches interleave."""
    gen = _gen(22)
    layer = Layer(gen, 512, 8, 1, 64, torch.float16)
    pools = [_pool(gen, 2, 24, 1, 64, torch.float16) for _ in range(2)]
    eager = [[c.clone() for c in cache] for cache, _ in pools]
    graphs = []
    for cache, table in pools:
        x, res = (torch.zeros((2, 1, 512), dtype=torch.float16, device="cuda") for _ in range(2))
        ids, pos, lens = _i32([0, 0]), _i32([[0], [0]]), _i32([0, 0])
        keep = [c.clone() for c in cache]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            layer(x, res, ids, pos, cache, table, lens)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = layer(x, res, ids, pos, cache, table, lens)
        for c, k in zip(cache, keep):
            c.copy_(k)
        graphs.append((g, x, res, ids, pos, lens, y))
    for i in range(40):
        for (g, x, res, ids, pos, lens, y), (cache, table), e in zip(graphs, pools, eager):
            x.copy_(torch.randn(x.shape, device="cuda", generator=gen))
            res.copy_(torch.randn(x.shape, device="cuda", generator=gen))
            ids.copy_(torch.randint(-1, 4, (2,), device="cuda", generator=gen))
            pos.copy_(_i32([[i], [i + 700]]))
            lens.copy_(_i32([i, i + 700]))
            g.replay()
            want = layer(x, res, ids, pos, e, table, lens)
            torch.cuda.synchronize()
            assert torch.equal(y, want) and all(torch.equal(a, c) for a, c in zip(cache, e))


def test_on_other_streams(cuda):
    """Calls in turn on two streams, each with data of its own, the workspaces from the allocator."""
    gen = _gen(23)
    sets = []
    for i in range(2):
        cache, table = _pool(gen, 4, 60, 1, 256, torch.bfloat16)
        q = torch.randn((4, 1, 8, 256), device="cuda", generator=gen).bfloat16()
        lens = _i32([3800, 3, 700, 64 + i])
        sets.append((q, *cache, table, lens, 0.06))
    wants = [w4a4.kv_attention(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i in range(16):
        with torch.cuda.stream(streams[i % 2]):
            got.append(w4a4.kv_attention(*sets[i % 2]))
    torch.cuda.synchronize()
    assert all(torch.equal(g, wants[i % 2]) for i, g in enumerate(got))


def test_refusals(cuda):
    gen = _gen(24)
    cache, table = _pool(gen, 2, 2, 1, 64, torch.float16)
    q = torch.zeros((2, 1, 2, 64), dtype=torch.float16, device="cuda")
    k, lens = q[:, :, :1], _i32([1, 1])

    def attend(q=q, cache=cache, table=table, lens=lens, **kw):
        return w4a4.kv_attention(q, *cache, table, lens, 0.1, **kw)

    def append(k=k, v=k, cache=cache, table=table, lens=lens, **kw):
        return w4a4.kv_append(k, v, *cache, table, lens, **kw)

    shared = [
        (dict(cache=[c.bfloat16() for c in cache]), "k_cache"), (dict(cache=[cache[0], cache[1][:1]]), "v_cache"),
        (dict(cache=[c.cpu() for c in cache]), "must be on"), (dict(table=table.long()), "block_table"), (dict(table=table[:1]), "block_table"),
        (dict(lens=lens.long()), "lens"), (dict(lens=lens[:1]), "lens"), (dict(lens=lens.cpu()), "must be on"),
        (dict(cache=[torch.zeros((6, 1, 64, 128), dtype=torch.float16, device="cuda")[..., ::2]] * 2), "contiguous"),
    ]
    for kw, text in shared + [(dict(q=q.float()), "float16 or bfloat16"), (dict(q=q[0]), "expects q"), (dict(q=q.bfloat16()), "k_cache"),
                              (dict(q_lens=lens.long()), "q_lens"), (dict(q=q[..., :32]), "head_dim")]:
        with pytest.raises(RuntimeError, match=text):
            attend(**kw)
    for kw, text in shared + [(dict(k=k.float()), "float16 or bfloat16"), (dict(v=k.bfloat16()), "one type"), (dict(k=k[:, :0]), "expects k and v"),
                              (dict(counts=lens[:1]), "counts")]:
        with pytest.raises(RuntimeError, match=text):
            append(**kw)
    for scaling in (float("nan"), float("inf")):
        with pytest.raises(RuntimeError, match="finite"):
            w4a4.kv_attention(q, *cache, table, lens, scaling)
    with pytest.raises(RuntimeError, match="multiple of the KV heads"):
        w4a4.kv_attention(torch.zeros((2, 1, 3, 64), dtype=torch.float16, device="cuda"), *w4a4.kv_cache(4, 2, 64, torch.float16, "cuda"),
                          table, lens, 0.1)
    with pytest.raises(RuntimeError, match="must not lie in the cache"):
        append(v=cache[0][:2, :, :1])
    with pytest.raises(RuntimeError, match="must not overlap"):
        append(cache=[cache[0], cache[0]])
    append(k=k[:, :0], v=k[:, :0])
    assert attend(q=q[:, :0]).shape == (2, 0, 2, 64)
    far = 1 << 32
    wide = k[:1].expand(far + 1, 1, 1, 64)
    with pytest.raises(RuntimeError, match="at most"):
        append(k=wide, v=wide, table=table[:1].expand(far + 1, 2), lens=lens[:1].expand(far + 1))
    with pytest.raises(RuntimeError, match="at most"):
        attend(table=table[:, :1].expand(2, far + 1))


@pytest.mark.filterwarnings("ignore:There is a performance drop")
def test_vmap(cuda):
    """One call a sample, the same results; what writes in place is refused there."""
    gen = _gen(26)
    cache, table = _pool(gen, 3, 2, 1, 64, torch.float16)
    q, k = (torch.randn((3, 2, n, 64), device="cuda", generator=gen).half() for n in (4, 1))
    pos, freq, lens = torch.arange(6, device="cuda").view(3, 2), torch.rand(32, device="cuda", generator=gen), _i32([70, 128, 3])
    got = torch.vmap(lambda q, k, p: w4a4.qk_norm_rope(q[None], k[None], k[0, 0], None, 1e-6, p[None], freq))(q, k, pos)
    for i in range(3):
        want = w4a4.qk_norm_rope(q[i:i + 1], k[i:i + 1], k[i, 0, 0], None, 1e-6, pos[i:i + 1], freq)
        assert all(torch.equal(a[i], b) for a, b in zip(got, want))
    got = torch.vmap(lambda q, t, n: w4a4.kv_attention(q[None], *cache, t[None], n[None], 0.1, return_lse=True))(q, table, lens)
    want = w4a4.kv_attention(q, *cache, table, lens, 0.1, return_lse=True)
    assert all(torch.equal(a[:, 0], b) for a, b in zip(got, want))
    with pytest.raises(RuntimeError):
        torch.vmap(lambda k, t, n: w4a4.kv_append(k[None], k[None], *cache, t[None], n[None]))(k, table, lens)


def test_dispatched_route(cuda):
    gen = _gen(25)
    cache, table = _pool(gen, 2, 3, 1, 64, torch.float16)
    q = torch.randn((2, 1, 4, 64), device="cuda", generator=gen).half()
    want = w4a4.kv_attention(q, *cache, table, _i32([70, 130]), 0.1, return_lse=True)
    got = torch.compile(lambda q: w4a4.kv_attention(q, *cache, table, _i32([70, 130]), 0.1, return_lse=True), fullgraph=True, backend="eager")(q)
    assert all(torch.equal(a, b) for a, b in zip(got, want))

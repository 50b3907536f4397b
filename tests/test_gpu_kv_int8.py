"""The 8-bit KV cache: the append bit for bit against its definition, the attention against 64 bits.

Tolerance of the attention.  The queries are held to 1 / 65024 of their row's maximum, so a logit
is within e = |scaling| * max|q| / 65024 * max_key sum|k| (a size: with a negative scaling the
signed product bounded nothing; plus fp32 roundings, 2^-20 of its
size); a probability is then within 2 e + 2^-19 |logit| relatively, the weights are rounded to fp16
(2^-11, and 2^-25 of the largest weight x value below fp16's normal range), the accumulation
adds 2^-18, and the output type half a step.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from pi05_fast.w4a4 import int8 as i8
from pi05_fast.w4a4 import kv_int8 as kv

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16]
PAGE = 64


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------ append
def _append_ref(x, codes, scale, table, lens, counts):
    """x [B, T, KVH, D] into codes [P, KVH, 64, D] and scale [P, KVH], numpy fp32 / exact products."""
    f32 = np.float32
    for b in range(x.shape[0]):
        have, count, at = int(lens[b]), int(counts[b]), 0
        while at < count:
            slot, o = divmod(have + at, PAGE)
            n = min(PAGE - o, count - at)
            page = int(table[b, slot]) if slot < table.shape[1] else -1
            if 0 <= page < codes.shape[0]:
                for h in range(x.shape[2]):
                    rows = x[b, at:at + n, h].astype(f32)
                    s0 = scale[page, h] if o else f32(0)
                    if np.isfinite(rows).all() and np.isfinite(s0):
                        s = max(s0, f32(f32(np.abs(rows).max() / f32(127)) + f32(1e-12)))
                        ratio, inv = f32(s0 / s), f32(f32(1) / s)
                        if s > s0:
                            codes[page, h] = np.rint(codes[page, h].astype(np.float64) * np.float64(ratio)) if o else 0
                        codes[page, h, o:o + n] = np.rint(rows.astype(np.float64) * np.float64(inv))
                        scale[page, h] = s
                    else:
                        scale[page, h] = np.nan
                        codes[page, h] = 0
            at += n


def _same(a, b):
    return bool(((a == b) | (np.isnan(a) & np.isnan(b))).all())


class Cache:
    """A pool with junk in it, and its mirror on the host."""

    def __init__(self, gen, b, table_pages, kvh, d, spare=3):
        n = b * table_pages + spare
        self.t = list(kv.int8_kv_cache(n, kvh, d, "cuda"))
        for c in self.t[:2]:
            c.copy_(torch.randint(-127, 128, c.shape, device="cuda", generator=gen, dtype=torch.int8))
        for s in self.t[2:]:
            s.fill_(123.0)
        self.table = torch.randperm(n, device="cuda", generator=gen)[: b * table_pages].to(torch.int32).view(b, table_pages)
        self.mirror()

    def mirror(self):
        self.kc, self.ks, self.vs = (self.t[i].cpu().numpy().copy() for i in (0, 2, 3))
        self.vc = self.t[1].transpose(2, 3).cpu().numpy().copy()

    def append(self, k, v, lens, counts=None):
        b, t = k.shape[:2]
        kv.int8_kv_append(k, v, *self.t, self.table, _i32(lens), counts=None if counts is None else _i32(counts))
        counts = [t] * b if counts is None else counts
        for x, codes, scale in ((k, self.kc, self.ks), (v, self.vc, self.vs)):
            _append_ref(x.float().cpu().numpy(), codes, scale, self.table.cpu().numpy(), lens, counts)
        self.check()

    def check(self):
        assert np.array_equal(self.t[0].cpu().numpy(), self.kc)
        assert np.array_equal(self.t[1].transpose(2, 3).cpu().numpy(), self.vc)
        assert _same(self.t[2].cpu().numpy(), self.ks) and _same(self.t[3].cpu().numpy(), self.vs)


def _kv(gen, b, t, kvh, d, dtype):
    return tuple((torch.randn((b, t, kvh, d), device="cuda", generator=gen)
                  * (torch.rand((b, t, kvh, 1), device="cuda", generator=gen) + 0.2)).to(dtype) for _ in range(2))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kvh,d", [(1, 256), (2, 128), (3, 64)])
@pytest.mark.parametrize("t,lens,counts", [
    (1, [0, 1, 63, 64], None), (1, [5, 0, 127, 100], [1, 0, 1, 1]), (3, [62, 63, 0, 10], None), (64, [0, 64, 1, 63], None),
    (65, [0, 0, 30, 64], [65, 1, 40, 64]), (130, [0, 7, 64, 65], [130, 121, 0, 63]), (7, [60, 61, 57, 58], [7, 3, 7, 6]),
])
def test_append_is_exact(cuda, t, lens, counts, kvh, d, dtype):
    gen = _gen(t * 7 + d)
    c = Cache(gen, 4, 4, kvh, d)
    c.append(*_kv(gen, 4, max(max(lens), 1), kvh, d, dtype), [0] * 4, lens)  # what is there already
    c.append(*_kv(gen, 4, t, kvh, d, dtype), lens, counts)


def test_append_token_by_token(cuda):
    """A page filled by single tokens of growing size keeps to its definition, and close to the values."""
    gen = _gen(3)
    c = Cache(gen, 2, 2, 1, 256)
    ks, vs = [], []
    for i in range(70):
        k, v = _kv(gen, 2, 1, 1, 256, torch.float16)
        k *= 1 + i / 16
        c.append(k, v, [i, i])
        ks.append(k)
        vs.append(v)
    k = torch.cat(ks, 1)[:, :64, 0].float()
    page = c.table[:, 0].long()
    got = c.t[0][page, 0].float() * c.t[2][page, 0][:, None, None]
    # every growth rounds the earlier codes by at most half a step of the new scale
    steps = torch.unique((k[0].abs().amax(-1)).cummax(0).values).numel()
    assert ((got - k).abs().amax() <= (steps + 1) * 0.5 * c.t[2][page, 0].max() * 1.001).item()


def test_append_drops_what_has_no_page(cuda):
    gen = _gen(4)
    c = Cache(gen, 3, 2, 2, 64)
    c.table[1, 1] = -1
    c.table[2, 0] = 10**6
    c.append(*_kv(gen, 3, 150, 2, 64, torch.float16), [0, 0, 0])  # 150 tokens on tables of 128
    c.append(*_kv(gen, 3, 5, 2, 64, torch.float16), [128, 1000, 126])
    c.append(*_kv(gen, 3, 5, 2, 64, torch.float16), [3, 3, 3], [0, 0, 0])
    # lengths and counts out of range are taken as the nearest in range
    k, v = _kv(gen, 3, 2, 2, 64, torch.float16)
    kv.int8_kv_append(k, v, *c.t, c.table, _i32([10, 10, 10]), counts=_i32([-5, -1, -2]))
    c.check()
    kv.int8_kv_append(k, v, *c.t, c.table, _i32([-7, 10, 10]), counts=_i32([99, 0, 0]))
    for x, codes, scale in ((k, c.kc, c.ks), (v, c.vc, c.vs)):
        _append_ref(x.float().cpu().numpy(), codes, scale, c.table.cpu().numpy(), [0, 10, 10], [2, 0, 0])
    c.check()


def test_append_nonfinite_and_strides(cuda):
    gen = _gen(5)
    c = Cache(gen, 2, 3, 2, 128)
    wide = torch.randn((2, 100, 3 * 2 * 128), device="cuda", generator=gen).half()
    k = wide[:, :, :256].view(2, 100, 2, 128)
    v = torch.randn((2, 2, 100, 128), device="cuda", generator=gen).half().transpose(1, 2)
    c.append(k, v, [0, 20])
    k1, v1 = _kv(gen, 2, 3, 2, 128, torch.float16)
    k1[0, 1, 0, 5] = float("inf")
    v1[1, 2, 1, 127] = float("nan")
    k1[1, 2] = float("nan")  # behind the count: not read
    c.append(k1, v1, [100, 120], [3, 2])
    c.append(*_kv(gen, 2, 2, 2, 128, torch.float16), [103, 122])
    # the next owner of a page starts afresh
    c.append(*_kv(gen, 2, 70, 2, 128, torch.float16), [0, 64])
    odd = torch.randn((2, 4, 2, 129), device="cuda", generator=gen).half()[..., 1:]
    c.append(odd, odd, [70, 100])


# ------------------------------------------------------------------ attention
def _pool(gen, b, table_pages, kvh, d, spread=True):
    n = b * table_pages + 2
    t = list(kv.int8_kv_cache(n, kvh, d, "cuda"))
    for c in t[:2]:
        c.copy_(torch.randn(c.shape, device="cuda", generator=gen).mul_(40).round_().clamp_(-127, 127).to(torch.int8))
    for s in t[2:]:
        s.copy_(torch.exp(torch.randn(s.shape, device="cuda", generator=gen) * (1.0 if spread else 0.0)) * 0.02)
    table = torch.randperm(n, device="cuda", generator=gen)[: b * table_pages].to(torch.int32).view(b, table_pages)
    return t, table


def _reference(q, cache, table, lens, scaling, causal, q_lens):
    """out, lse and a bound on the out error (float64)."""
    kc, vc, ks, vs = cache
    b, t, h, d = q.shape
    kvh = kc.size(1)
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    lse = torch.full((b, t, h), float("-inf"), dtype=torch.float64, device="cuda")
    ltol = torch.zeros_like(lse)
    for i in range(b):
        n, ql = min(max(int(lens[i]), 0), table.size(1) * PAGE), t if q_lens is None else min(max(int(q_lens[i]), 0), t)
        ids = table[i].long()
        ok = ((ids >= 0) & (ids < kc.size(0))).repeat_interleave(PAGE)[:n]
        ids = ids.clamp(0, kc.size(0) - 1)
        for g in range(kvh):
            k = (kc[ids, g].double() * ks[ids, g].double()[:, None, None]).reshape(-1, d)[:n]
            v = (vc[ids, g].double() * vs[ids, g].double()[:, None, None]).transpose(1, 2).reshape(-1, d)[:n]
            for hh in range(g * (h // kvh), (g + 1) * (h // kvh)):
                for j in range(ql) if causal else [slice(0, ql)]:
                    m = min(max(n - ql + j + 1, 0), n) if causal else n
                    see = ok[:m]
                    if not see.any() or (not causal and ql == 0):
                        continue
                    rows = q[i, j:j + 1, hh] if causal else q[i, j, hh]
                    qq = rows.double()
                    z = (qq @ k[:m].t().contiguous() * scaling)[:, see]
                    p = torch.softmax(z, -1)
                    vv = v[:m][see]
                    where = (i, slice(j, j + 1), hh) if causal else (i, j, hh)
                    out[where] = p @ vv
                    lse[where] = torch.logsumexp(z, -1)
                    e = (abs(scaling) * qq.abs().amax(-1) / 65024 * k[:m][see].abs().sum(-1).max())[:, None]
                    rel = 2 * e + 2.0**-19 * z.abs().amax(-1, keepdim=True) + 2.0**-11 + 2.0**-18
                    tol[where] = rel * (p @ vv.abs()) + m * 2.0**-25 * vv.abs().max()
                    ltol[where] = (e + 2.0**-19 * z.abs().amax(-1, keepdim=True) + 1e-5)[:, 0]
    return out, lse, tol + (torch.finfo(q.dtype).eps / 2) * out.abs() * 1.001 + 2.0**-25, ltol


def _check_attention(q, cache, table, lens, scaling, causal=True, q_lens=None):
    li = _i32(lens)
    qi = None if q_lens is None else _i32(q_lens)
    got, lse = kv.int8_kv_attention(q, *cache, table, li, scaling, causal=causal, q_lens=qi, return_lse=True)
    want, wlse, tol, ltol = _reference(q, cache, table, lens, scaling, causal, q_lens)
    assert torch.isfinite(got).all()
    over = ((got.double() - want).abs() / tol).max().item()
    assert over <= 1
    inf = torch.isinf(wlse)
    assert torch.equal(inf, torch.isinf(lse)) and ((lse.double() - wlse).abs() <= ltol + 2e-7 * wlse.abs())[~inf].all()
    assert not got[inf].any()
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("h,kvh,d", [(8, 1, 256), (6, 2, 128), (5, 5, 64), (40, 2, 64), (1, 1, 256)])
@pytest.mark.parametrize("lens,t", [([1], 1), ([0, 64, 65], 1), ([63, 300, 1000, 7], 1), ([130, 5, 64], 5), ([70, 200], 70)])
def test_attention(cuda, lens, t, h, kvh, d, dtype):
    gen = _gen(t + h + d)
    b = len(lens)
    cache, table = _pool(gen, b, (max(lens) + 63) // 64 + 1, kvh, d)
    q = (torch.randn((b, t, h, d), device="cuda", generator=gen) * 1.5).to(dtype)
    for causal in (True, False):
        _check_attention(q, cache, table, lens, d**-0.5, causal)


@pytest.mark.parametrize("h,kvh,d", [(8, 1, 256), (4, 4, 128)])
def test_attention_ragged_queries(cuda, h, kvh, d):
    """Padding queries, sequences shorter than their queries, and none at all: zeros."""
    gen = _gen(11)
    cache, table = _pool(gen, 5, 5, kvh, d)
    q = torch.randn((5, 40, h, d), device="cuda", generator=gen).half()
    q[2] = float("nan")  # a sequence without queries
    q[3, 7:] = float("inf")  # behind the last query
    for causal in (True, False):
        got, lse = kv.int8_kv_attention(q, *cache, table, _i32([300, 10, 64, 200, 0]), 0.06, causal=causal,
                                        q_lens=_i32([40, 25, 0, 7, 33]), return_lse=True)
        q0 = torch.where(torch.isfinite(q), q, torch.zeros_like(q))
        want, wlse, tol, _ = _reference(q0, cache, table, [300, 10, 64, 200, 0], 0.06, causal, [40, 25, 0, 7, 33])
        assert ((got.double() - want).abs() <= tol).all()
        assert torch.equal(torch.isinf(wlse), torch.isinf(lse))


def test_attention_table_edges(cuda):
    """Lengths past the table, entries that name no page, sequences that share pages."""
    gen = _gen(12)
    cache, table = _pool(gen, 4, 3, 1, 128)
    table[1] = table[0]
    table[2, 1] = -1
    table[3, 0] = 10**9
    q = torch.randn((4, 2, 4, 128), device="cuda", generator=gen).half()
    _check_attention(q, cache, table, [192, 100, 192, 150], 0.09)
    _check_attention(q, cache, table, [10**6, -3, 70, 30], 0.09, causal=False)
    wide = torch.full((4, 9), -1, dtype=torch.int32, device="cuda")
    wide[:, 2:5] = table
    a = kv.int8_kv_attention(q, *cache, wide[:, 2:5], _i32([192, 100, 50, 150]), 0.09)
    assert torch.equal(a, kv.int8_kv_attention(q, *cache, table, _i32([192, 100, 50, 150]), 0.09))


def test_attention_hidden_junk(cuda):
    """What no query sees has no effect: codes behind the last token, scales of pages not reached
    (NaN and infinities among them), pages behind the causal edge."""
    gen = _gen(13)
    cache, table = _pool(gen, 2, 4, 1, 256)
    lens = [100, 129]
    for t in (1, 30):
        q = torch.randn((2, t, 8, 256), device="cuda", generator=gen).half()
        want = _check_attention(q, cache, table, lens, 0.06)
        dirty = [c.clone() for c in cache]
        for b, n in enumerate(lens):
            page = int(table[b, n // 64])
            dirty[0][page, :, n % 64:] = 127
            dirty[1][page, :, :, n % 64:] = -127
            for s in dirty[2:]:
                s[table[b, n // 64 + 1:].long()] = float("nan") if b else float("inf")
        assert torch.equal(kv.int8_kv_attention(q, *dirty, table, _i32(lens), 0.06), want)
    # the last page's scales NaN: the queries before it do not see that
    q = torch.randn((2, 30, 8, 256), device="cuda", generator=gen).half()
    want = kv.int8_kv_attention(q, *cache, table, _i32(lens), 0.06)
    for i in (2, 3):
        dirty = [c.clone() for c in cache]
        dirty[i][table[1, 2].long()] = float("nan")
        got = kv.int8_kv_attention(q, *dirty, table, _i32(lens), 0.06)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1, :-1], want[1, :-1]) and torch.isnan(got[1, -1]).all()


def test_attention_extremes(cuda):
    """Pages whose scales differ by ten orders of magnitude, zero values, peaked and flat rows."""
    gen = _gen(14)
    cache, table = _pool(gen, 2, 10, 1, 256, spread=False)
    cache[3][table[0, 1].long()] = 1e-12
    cache[3][table[0, 2].long()] = 300.0
    cache[3][table[1, 0].long()] = 0.0
    cache[2][table[1, 3].long()] = 0.0
    q = torch.randn((2, 3, 8, 256), device="cuda", generator=gen).half()
    for scaling in (0.0, 0.0625, 1.0, -0.0625):
        _check_attention(q, cache, table, [640, 600], scaling)
    _check_attention(q * 0, cache, table, [640, 600], 0.0625)
    _check_attention((q * 3000).clamp(-60000, 60000), cache, table, [640, 600], 1e-5)
    b = torch.randn((2, 3, 8, 256), device="cuda", generator=gen).bfloat16()
    _check_attention(b * 1e30, cache, table, [640, 600], 6e-32)
    _check_attention(b * 1e-30, cache, table, [640, 600], 6e28)
    q[1, 2, 3, 100] = float("nan")
    got = kv.int8_kv_attention(q, *cache, table, _i32([640, 600]), 0.0625)
    assert torch.isnan(got[1, 2, 3]).all()
    got[1, 2, 3] = 0
    assert torch.isfinite(got).all()


def test_attention_long(cuda):
    gen = _gen(15)
    cache, table = _pool(gen, 2, 520, 1, 256)
    q = torch.randn((2, 1, 8, 256), device="cuda", generator=gen).half()
    _check_attention(q, cache, table, [33000, 1], 0.0625)
    _check_attention(q, cache, table, [33280, 20000], 0.0, causal=False)
    q = torch.randn((2, 300, 8, 256), device="cuda", generator=gen).half()
    _check_attention(q, cache, table, [5000, 333], 0.0625, causal=False)


def test_attention_pool_past_4_gib(cuda):
    """Pages whose codes lie behind 2^32 bytes."""
    gen = _gen(16)
    small, _ = _pool(gen, 1, 4, 1, 256)
    n = 280000
    kc, vc, ks, vs = kv.int8_kv_cache(n, 1, 256, "cuda")
    ids = torch.tensor([n - 1, 270000, 5, n - 2], device="cuda")
    for big, part in zip((kc, vc, ks, vs), small):
        big[ids] = part[:4]
    q = torch.randn((1, 2, 8, 256), device="cuda", generator=gen).half()
    a = kv.int8_kv_attention(q, kc, vc, ks, vs, ids.to(torch.int32).view(1, 4), _i32([250]), 0.06)
    assert torch.equal(a, kv.int8_kv_attention(q, *small, _i32([[0, 1, 2, 3]]), _i32([250]), 0.06))
    k, v = _kv(gen, 1, 3, 1, 256, torch.float16)
    kv.int8_kv_append(k, v, kc, vc, ks, vs, ids.to(torch.int32).view(1, 4), _i32([190]))
    kv.int8_kv_append(k, v, *small, _i32([[0, 1, 2, 3]]), _i32([190]))
    for big, part in zip((kc, vc, ks, vs), small):
        assert torch.equal(big[ids], part[:4])


def test_query_strides(cuda):
    gen = _gen(17)
    cache, table = _pool(gen, 3, 4, 1, 256)
    wide = torch.randn((3, 6, 2560), device="cuda", generator=gen).half()
    q = wide[:, :, :2048].view(3, 6, 8, 256)
    lens = _i32([200, 65, 6])
    want = kv.int8_kv_attention(q.contiguous(), *cache, table, lens, 0.06)
    assert torch.equal(kv.int8_kv_attention(q, *cache, table, lens, 0.06), want)
    turned = q.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(kv.int8_kv_attention(turned, *cache, table, lens, 0.06), want)
    odd = torch.zeros((3, 6, 8, 257), device="cuda", dtype=torch.float16)
    odd[..., 1:] = q
    assert torch.equal(kv.int8_kv_attention(odd[..., 1:], *cache, table, lens, 0.06), want)
    one = kv.int8_kv_attention(q[:, :1, :1].expand(3, 6, 8, 256), *cache, table, lens, 0.06)
    assert torch.equal(one, kv.int8_kv_attention(q[:, :1, :1].expand(3, 6, 8, 256).contiguous(), *cache, table, lens, 0.06))


def _reference_many(q, cache, table, lens, scaling, causal, q_lens):
    """_reference with all tokens of a head at once, and the same bounds."""
    kc, vc, ks, vs = cache
    b, t, h, d = q.shape
    kvh = kc.size(1)
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    lse = torch.full((b, t, h), float("-inf"), dtype=torch.float64, device="cuda")
    for i in range(b):
        n, ql = min(max(lens[i], 0), table.size(1) * PAGE), min(max(q_lens[i], 0), t)
        if n == 0 or ql == 0:
            continue
        ids = table[i].long()
        ok = ((ids >= 0) & (ids < kc.size(0))).repeat_interleave(PAGE)[:n]
        ids = ids.clamp(0, kc.size(0) - 1)
        at = torch.arange(n, device="cuda")
        last = n - ql + torch.arange(ql, device="cuda") if causal else torch.full((ql,), n, device="cuda")
        see = ok & (at <= last[:, None])
        some = see.any(-1)
        for g in range(kvh):
            k = (kc[ids, g].double() * ks[ids, g].double()[:, None, None]).reshape(-1, d)[:n].nan_to_num(0, 0, 0) * ok[:, None]
            v = (vc[ids, g].double() * vs[ids, g].double()[:, None, None]).transpose(1, 2).reshape(-1, d)[:n].nan_to_num(0, 0, 0) * ok[:, None]
            for hh in range(g * (h // kvh), (g + 1) * (h // kvh)):
                qq = q[i, :ql, hh].double()
                z = (qq @ k.t().contiguous() * scaling).masked_fill(~see, float("-inf"))
                p = torch.softmax(z, -1).nan_to_num(0)
                top = z.masked_fill(~see, 0).abs().amax(-1, keepdim=True)
                e = (abs(scaling) * qq.abs().amax(-1) / 65024 * k.abs().sum(-1).max())[:, None]
                out[i, :ql, hh] = p @ v
                lse[i, :ql, hh] = torch.logsumexp(z, -1)
                tol[i, :ql, hh] = some[:, None] * ((2 * e + 2.0**-19 * top + 2.0**-11 + 2.0**-18) * (p @ v.abs())
                                                   + n * 2.0**-25 * v.abs().max())
    return out, lse, tol + (torch.finfo(q.dtype).eps / 2) * out.abs() * 1.001 + 2.0**-25


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,t,h,kvh,d,pages", [
    (4, 300, 8, 1, 256, 3), (4, 300, 8, 1, 256, 20), (1, 300, 8, 1, 256, 64), (4, 1100, 2, 2, 256, 2),
    (4, 800, 8, 1, 128, 3), (4, 700, 6, 2, 128, 30), (5, 451, 8, 2, 64, 2), (4, 1501, 8, 2, 64, 4), (4, 50, 32, 8, 128, 32),
])
def test_attention_of_chunks(cuda, b, t, h, kvh, d, pages, dtype):
    """More rows than one round of small workgroups: whole and ragged chunks, a sequence shorter than its queries, an
    empty one, junk behind the last token and queries, a page that is none."""
    gen = _gen(t + pages)
    cache, table = _pool(gen, b, pages, kvh, d)
    q = (torch.randn((b, t, h, d), device="cuda", generator=gen) * 1.5).to(dtype)
    lens = [pages * PAGE - 3, pages * PAGE + 9, 70, 0, 65][:b]
    q_lens = [t, t - 40, min(t, 100), t, 7][:b]
    for i, n in enumerate(lens):
        if n < (pages - 1) * PAGE:
            for s in cache[2:]:
                s[table[i, n // PAGE + 1:].long()] = float("nan")
        q[i, q_lens[i]:] = float("nan")
    if b > 1:
        table[1, 1] = -1
    for causal in (True, False):
        got, lse = kv.int8_kv_attention(q, *cache, table, _i32(lens), d**-0.5, causal=causal, q_lens=_i32(q_lens), return_lse=True)
        want, wlse, tol = _reference_many(q, cache, table, lens, d**-0.5, causal, q_lens)
        assert ((got.double() - want).abs() / tol).max().item() <= 1
        inf = torch.isinf(wlse)
        assert torch.equal(inf, torch.isinf(lse)) and not got[inf].any()
        assert ((lse.double() - wlse).abs() <= 1e-3 + 1e-3 * wlse.abs())[~inf].all()


def test_chunks_of_other_strides(cuda):
    """Queries that are a part of a product's output, and results that do not depend on where they lie."""
    gen = _gen(23)
    cache, table = _pool(gen, 4, 4, 1, 256)
    wide = torch.randn((4, 301, 2560), device="cuda", generator=gen).half()
    q = wide[:, 1:, :2048].view(4, 300, 8, 256)
    lens = _i32([250, 256, 3, 190])
    want = kv.int8_kv_attention(q.contiguous(), *cache, table, lens, 0.06)
    assert torch.equal(kv.int8_kv_attention(q, *cache, table, lens, 0.06), want)
    turned = q.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(kv.int8_kv_attention(turned, *cache, table, lens, 0.06), want)


def test_joined_with_other_keys(cuda):
    """Two halves of a cache joined by their lse are the whole."""
    gen = _gen(18)
    cache, table = _pool(gen, 2, 6, 1, 256, spread=False)
    q = torch.randn((2, 4, 8, 256), device="cuda", generator=gen).half()
    parts = [kv.int8_kv_attention(q, *cache, tb.contiguous(), _i32(n), 0.06, causal=False, return_lse=True)
             for tb, n in ((table[:, :3], [192, 192]), (table[:, 3:], [180, 20]))]
    whole, lse = kv.int8_kv_attention(q, *cache, table, _i32([372, 212]), 0.06, causal=False, return_lse=True)
    both = torch.logaddexp(parts[0][1], parts[1][1])
    joined = sum(o.float() * torch.exp(l - both)[..., None] for o, l in parts)
    assert (both - lse).abs().max() < 1e-4
    v = 127 * 0.02
    assert (joined - whole.float()).abs().max() < 2.0**-9 * v + 2.0**-10 * v  # two fp16 parts, one whole, weights of 2^-11


# ------------------------------------------------------------------ the operators together
def _step(x, res, p, cache, table, lens, dtype):
    """The 8-bit attention half of a layer for T new tokens of each sequence."""
    b, t, width = x.shape
    q8, s, h = i8.add_rms_norm_int8(x, res, p["norm"], 1e-6)
    qkv = i8.int8_gemm(q8, s, *p["qkv"], out_dtype=dtype)
    hd = p["d"]
    q = qkv[..., : p["h"] * hd].view(b, t, p["h"], hd)
    k = qkv[..., p["h"] * hd: (p["h"] + 1) * hd].view(b, t, 1, hd)
    v = qkv[..., (p["h"] + 1) * hd:].view(b, t, 1, hd)
    kv.int8_kv_append(k, v, *cache, table, lens)
    att = kv.int8_kv_attention(q, *cache, table, lens + t, hd**-0.5)
    a8, sa = i8.quantize_int8(att.view(b, t, -1))
    return i8.int8_gemm(a8, sa, *p["o"], residual=h, out_dtype=dtype), (q, k, v, att, h)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_half_of_a_layer(cuda, dtype):
    """Norm, QKV, append, attention and o for a prompt in two chunks and then single tokens: each step against
    64 bits from the step's own inputs, and the cache against the definition of its append."""
    gen = _gen(19)
    width, heads, d, b = 512, 4, 128, 3
    p = {"norm": (torch.randn(width, device="cuda", generator=gen) * 0.1).to(dtype), "h": heads, "d": d,
         "qkv": i8.quantize_int8((torch.randn(((heads + 2) * d, width), device="cuda", generator=gen) * 0.05).to(dtype)),
         "o": i8.quantize_int8((torch.randn((width, heads * d), device="cuda", generator=gen) * 0.05).to(dtype))}
    c = Cache(gen, b, 4, 1, d)
    have = 0
    for t in (90, 37, 1, 1, 1):
        x, res = (torch.randn((b, t, width), device="cuda", generator=gen).to(dtype) for _ in range(2))
        lens = _i32([have] * b)
        y, (q, k, v, att, h) = _step(x, res, p, c.t, c.table, lens, dtype)
        for xx, codes, scale in ((k, c.kc, c.ks), (v, c.vc, c.vs)):
            _append_ref(xx.float().cpu().numpy(), codes, scale, c.table.cpu().numpy(), [have] * b, [t] * b)
        c.check()
        have += t
        want, _, tol, _ = _reference(q, c.t, c.table, [have] * b, d**-0.5, True, None)
        assert ((att.double() - want).abs() <= tol).all()
        a8, sa = i8.quantize_int8(att.reshape(b * t, -1))
        prod = (a8.double() @ p["o"][0].double().t().contiguous()) * sa.double()[:, None] * p["o"][1].double()
        ref = prod + h.reshape(b * t, -1).double()
        bound = 2.0**-20 * (prod.abs() + h.reshape(b * t, -1).double().abs()) + torch.finfo(dtype).eps / 2 * 1.001 * ref.abs() + 2.0**-25
        assert ((y.reshape(b * t, -1).double() - ref).abs() <= bound).all()


def test_captured_decode_steps(cuda):
    """A captured step, replayed with moving lengths, does what the eager steps do; two graphs on their own caches
    interleave."""
    gen = _gen(20)
    width, heads, d, b = 512, 8, 64, 2
    p = {"norm": torch.zeros(width, dtype=torch.float16, device="cuda"), "h": heads, "d": d,
         "qkv": i8.quantize_int8((torch.randn(((heads + 2) * d, width), device="cuda", generator=gen) * 0.05).half()),
         "o": i8.quantize_int8((torch.randn((width, heads * d), device="cuda", generator=gen) * 0.05).half())}
    caches = [Cache(gen, b, 24, 1, d) for _ in range(2)]
    eager = [[t.clone() for t in c.t] for c in caches]
    graphs = []
    for c in caches:
        x, res, lens = torch.zeros((b, 1, width), dtype=torch.float16, device="cuda"), torch.zeros((b, 1, width), dtype=torch.float16, device="cuda"), _i32([0, 0])
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        keep = [t.clone() for t in c.t]
        with torch.cuda.stream(side):
            _step(x, res, p, c.t, c.table, lens, torch.float16)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y, _ = _step(x, res, p, c.t, c.table, lens, torch.float16)
        for t, k in zip(c.t, keep):
            t.copy_(k)
        graphs.append((g, x, res, lens, y))
    for i in range(66):
        for (g, x, res, lens, y), c, e in zip(graphs, caches, eager):
            xi, ri = (torch.randn((b, 1, width), device="cuda", generator=gen).half() for _ in range(2))
            x.copy_(xi)
            res.copy_(ri)
            lens.copy_(_i32([i, i + 3]))
            g.replay()
            want, _ = _step(xi, ri, p, e, c.table, _i32([i, i + 3]), torch.float16)
            if i % 8 == 0 or i > 62:
                torch.cuda.synchronize()
                assert torch.equal(y, want)
                assert all(torch.equal(a, b2) for a, b2 in zip(c.t[:2], e[:2]))


def test_on_another_stream(cuda):
    gen = _gen(21)
    cache, table = _pool(gen, 4, 30, 1, 256)
    q = torch.randn((4, 1, 8, 256), device="cuda", generator=gen).half()
    lens = _i32([1900, 3, 700, 64])
    want = kv.int8_kv_attention(q, *cache, table, lens, 0.06)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i in range(10):
        with torch.cuda.stream(streams[i % 2]):
            got.append(kv.int8_kv_attention(q, *cache, table, lens, 0.06))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_refusals_on_the_gpu(cuda):
    gen = _gen(22)
    cache, table = _pool(gen, 2, 2, 1, 64)
    q = torch.zeros((2, 1, 2, 64), dtype=torch.float16, device="cuda")
    k = q[:, :, :1]
    lens = _i32([1, 1])

    def attend(q=q, cache=cache, table=table, lens=lens, **kw):
        return kv.int8_kv_attention(q, *cache, table, lens, 0.1, **kw)

    def append(k=k, v=k, cache=cache, table=table, lens=lens, **kw):
        return kv.int8_kv_append(k, v, *cache, table, lens, **kw)

    def swapped(i, t):
        return [t if j == i else c for j, c in enumerate(cache)]

    shared = [
        (dict(cache=swapped(0, cache[0].to(torch.uint8))), "k_cache"), (dict(cache=swapped(1, cache[1][:1])), "v_cache"),
        (dict(cache=swapped(2, cache[2].half())), "k_scale"), (dict(cache=swapped(3, cache[3][:1])), "v_scale"),
        (dict(cache=swapped(2, cache[2].cpu())), "must be on"), (dict(table=table.long()), "block_table"),
        (dict(table=table[:1]), "block_table"), (dict(lens=lens.long()), "lens"), (dict(lens=lens[:1]), "lens"),
        (dict(lens=lens.cpu()), "must be on"),
        (dict(cache=swapped(1, torch.zeros((cache[1].size(0), 1, 64, 128), dtype=torch.int8, device="cuda")[..., ::2])), "contiguous"),
    ]
    for kw, text in shared + [(dict(q=q.float()), "float16 or bfloat16"), (dict(q=q[0]), "expects q"),
                              (dict(q_lens=lens.long()), "q_lens"), (dict(q=q[..., :32]), "head_dim")]:
        with pytest.raises(RuntimeError, match=text):
            attend(**kw)
    for kw, text in shared + [(dict(k=k.float()), "float16 or bfloat16"), (dict(v=k.bfloat16()), "one type"),
                              (dict(k=k[:, :0]), "expects k and v"), (dict(counts=lens[:1]), "counts")]:
        with pytest.raises(RuntimeError, match=text):
            append(**kw)
    with pytest.raises(RuntimeError, match="multiple of the KV heads"):
        kv.int8_kv_attention(torch.zeros((2, 1, 3, 64), dtype=torch.float16, device="cuda"),
                             *kv.int8_kv_cache(4, 2, 64, "cuda"), table, lens, 0.1)
    append(k=k[:, :0], v=k[:, :0])
    assert attend(q=q[:, :0]).shape == (2, 0, 2, 64)
    assert not attend(cache=kv.int8_kv_cache(0, 1, 64, "cuda"), table=table[:, :0]).any()


def test_dispatched_route(cuda):
    gen = _gen(23)
    cache, table = _pool(gen, 2, 3, 1, 64)
    q = torch.randn((2, 1, 4, 64), device="cuda", generator=gen).half()
    k, v = _kv(gen, 2, 1, 1, 64, torch.float16)
    other = [c.clone() for c in cache]
    lens = _i32([70, 64])

    def step(q, k, v, kc, vc, ks, vs):
        kv.int8_kv_append(k, v, kc, vc, ks, vs, table, lens)
        return kv.int8_kv_attention(q, kc, vc, ks, vs, table, lens + 1, 0.1)

    want = step(q, k, v, *cache)
    got = torch.compile(step, fullgraph=True, backend="eager")(q, k, v, *other)
    assert torch.equal(got, want) and all(torch.equal(a, b) for a, b in zip(cache, other))

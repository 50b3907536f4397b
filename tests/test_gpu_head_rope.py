"""Head norms and rotary positions against 64 bits, and what they write into a 16-bit KV cache.

Tolerance: the sum of squares of D <= 512 elements is at most 2^-19 off relatively (16 sums in a lane and 5
across them, of 2^-24, twice over), its root half of that, the root, the quotient and the products
2^-22; sine and cosine are 2^-21 off (an angle of at most half a turn rounded to 24 bits: pi 2^-25, and two steps
of a result below 1).  So a rotated element is within 2^-19 (|f1| + |f2|), and half a step of its type.
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


def _freq(rot, theta=10000.0):
    j = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    return (theta ** (-2 * j / max(rot, 1))).float()


def _ref(x, w, eps, pos, freq, unit_offset=True, interleaved=False, axes=None):
    """(result, bound) in 64 bits."""
    f = x.double()
    if w is not None:
        f = f / torch.sqrt((f * f).mean(-1, keepdim=True) + eps) * (w.double() + (1 if unit_offset else 0))
    out, mag = f.clone(), f.abs()
    for j in range(freq.numel()):
        i0, i1 = (2 * j, 2 * j + 1) if interleaved else (j, j + freq.numel())
        p = pos if pos.dim() == 2 else pos[0 if axes is None else axes[j]]
        angle = (p.double() * freq[j].double())[:, :, None]
        c, s = torch.cos(angle), torch.sin(angle)
        out[..., i0] = f[..., i0] * c - f[..., i1] * s
        out[..., i1] = f[..., i1] * c + f[..., i0] * s
        mag[..., i0] = mag[..., i1] = f[..., i0].abs() + f[..., i1].abs()
    return out, mag * 2.0**-19 + torch.finfo(x.dtype).eps / 2 * 1.001 * out.abs() + 2.0**-25


def _check(got, x, *args, **kw):
    want, tol = _ref(x, *args, **kw)
    assert got.dtype == x.dtype and got.shape == x.shape and got.is_contiguous()
    assert ((got.double() - want).abs() <= tol).all(), ((got.double() - want).abs() / tol).max().item()


def _heads(gen, b, t, h, kvh, d, dtype):
    joined = torch.randn((b, t, (h + 2 * kvh) * d), device="cuda", generator=gen)
    joined[..., ::97] *= 20
    x = joined.to(dtype).view(b, t, h + 2 * kvh, d)
    return x[:, :, :h], x[:, :, h:h + kvh], x[:, :, h + kvh:]


def _weights(gen, d, dtype):
    return [(torch.randn(d, device="cuda", generator=gen) * 0.2).to(dtype) for _ in range(2)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("h,kvh,d,rot", [(8, 1, 256, 256), (32, 8, 128, 128), (8, 8, 64, 64), (5, 5, 80, 80), (12, 3, 96, 64),
                                         (4, 1, 512, 512), (7, 7, 112, 16), (1, 1, 16, 16), (3, 1, 32, 0), (70, 2, 128, 96)])
@pytest.mark.parametrize("b,t", [(1, 1), (3, 7), (2, 300)])
def test_heads(cuda, b, t, h, kvh, d, rot, dtype):
    gen = _gen(b + t + h + d)
    q, k, _ = _heads(gen, b, t, h, kvh, d, dtype)
    qw, kw = _weights(gen, d, dtype)
    pos = torch.randint(0, 9000, (b, t), device="cuda", generator=gen).to(torch.int32)
    for interleaved in (False, True):
        qo, ko = w4a4.qk_norm_rope(q, k, qw, kw, 1e-6, pos, _freq(rot), interleaved=interleaved)
        _check(qo, q, qw, 1e-6, pos, _freq(rot), interleaved=interleaved)
        _check(ko, k, kw, 1e-6, pos, _freq(rot), interleaved=interleaved)


def test_forms_of_the_norm(cuda):
    gen = _gen(2)
    q, k, _ = _heads(gen, 2, 5, 8, 1, 256, torch.float16)
    qw, kw = _weights(gen, 256, torch.float16)
    pos = _i32([[0, 1, 2, 3, 4], [-5, 100, 7, 8, 1 << 20]])
    for a, b, unit, eps in ((None, None, True, 0.0), (qw, None, True, 1e-6), (None, kw, False, 1e-2), (qw, kw, False, 0.0)):
        qo, ko = w4a4.qk_norm_rope(q, k, a, b, eps, pos, _freq(256), unit_offset=unit)
        _check(qo, q, a, eps, pos, _freq(256), unit)
        _check(ko, k, b, eps, pos, _freq(256), unit)
    # without a norm and at position 0, as they were
    qo, ko = w4a4.qk_norm_rope(q, k, None, None, 0.0, pos * 0, _freq(256))
    assert torch.equal(qo, q) and torch.equal(ko, k)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ptype", [torch.int32, torch.int64])
def test_axes(cuda, dtype, ptype):
    gen = _gen(3)
    q, k, _ = _heads(gen, 2, 33, 6, 2, 128, dtype)
    qw, kw = _weights(gen, 128, dtype)
    for count, axes in ((1, None), (3, w4a4.rope_axes((16, 24, 24))), (3, [j % 3 for j in range(64)]), (2, [1] * 64),
                        (4, [(j * 7) % 4 for j in range(64)])):
        pos = torch.randint(0, 5000, (count, 2, 33), device="cuda", generator=gen).to(ptype)
        for interleaved in (False, True):
            qo, ko = w4a4.qk_norm_rope(q, k, qw, kw, 1e-6, pos, _freq(128), interleaved=interleaved, axes=axes)
            _check(qo, q, qw, 1e-6, pos, _freq(128), interleaved=interleaved, axes=axes)
            _check(ko, k, kw, 1e-6, pos, _freq(128), interleaved=interleaved, axes=axes)


def test_far_positions(cuda):
    """Positions whose angles 32 bits do not hold."""
    gen = _gen(4)
    q, k, _ = _heads(gen, 1, 6, 2, 1, 64, torch.float16)
    pos = torch.tensor([[2**31 - 1, -(2**31), 2**24 + 1, 123456789, 999999, 2**40 + 3]], device="cuda")
    # 2^40 * 2^-52 of a turn
    qo, ko = w4a4.qk_norm_rope(q, k, None, None, 0.0, pos, _freq(64))
    want, tol = _ref(q, None, 0.0, pos, _freq(64))
    assert ((qo.double() - want).abs() <= tol + q.double().abs().max() * 2.0**-10 * (pos.abs() > 2**39)[..., None, None]).all()
    near = pos[:, :5].to(torch.int32)
    a, _ = w4a4.qk_norm_rope(q[:, :5], k[:, :5], None, None, 0.0, near, _freq(64))
    assert torch.equal(a, qo[:, :5])


def test_strides(cuda):
    gen = _gen(5)
    q, k, _ = _heads(gen, 3, 9, 4, 2, 64, torch.float16)
    pos = torch.arange(9, device="cuda", dtype=torch.int32)[None].expand(3, 9)
    want = w4a4.qk_norm_rope(q.contiguous(), k.contiguous(), None, None, 0.0, pos.contiguous(), _freq(64))
    odd = torch.zeros((3, 9, 4, 65), device="cuda", dtype=torch.float16)
    odd[..., 1:] = q
    wide = torch.zeros((9, 3), device="cuda", dtype=torch.int32).t()
    wide.copy_(pos)
    qw = torch.ones(65, device="cuda", dtype=torch.float16)[1:]
    for qq, pp in ((q, pos), (q.transpose(1, 2).contiguous().transpose(1, 2), wide), (odd[..., 1:], pos)):
        got = w4a4.qk_norm_rope(qq, k, None, None, 0.0, pp, _freq(64))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    a, _ = w4a4.qk_norm_rope(q, k, qw, None, 1e-6, pos, _freq(64))
    assert torch.equal(a, w4a4.qk_norm_rope(q, k, qw.clone(), None, 1e-6, pos, _freq(64))[0])
    one = w4a4.qk_norm_rope(q[:, :, :1].expand(3, 9, 4, 64), k, None, None, 0.0, pos, _freq(128)[:32])
    assert torch.equal(one[0], w4a4.qk_norm_rope(q[:, :, :1].expand(3, 9, 4, 64).contiguous(), k, None, None, 0.0, pos, _freq(128)[:32])[0])


def test_range_of_the_norm(cuda):
    """Heads whose squares leave fp32's range, zeros, and heads that are not finite, which leave the others alone."""
    gen = _gen(6)
    x = torch.randn((2, 3, 4, 128), device="cuda", generator=gen).bfloat16()
    k = x[:, :, :1]
    w = _weights(gen, 128, torch.bfloat16)[0]
    pos = _i32([[1, 2, 3], [4, 5, 6]])
    for scale in (1e30, 1e-25, 3e37, 1e-38):
        for eps in (0.0, 1e-6):
            got, _ = w4a4.qk_norm_rope(x * scale, k, w, None, eps, pos, _freq(128))
            _check(got, x * scale, w, eps, pos, _freq(128))
    got, _ = w4a4.qk_norm_rope(x * 0, k, w, None, 1e-6, pos, _freq(128))
    assert not got.any()
    bad = x.clone()
    bad[0, 1, 2, 5] = float("inf")
    bad[1, 0, 0, 7] = float("nan")
    got, _ = w4a4.qk_norm_rope(bad, k, w, None, 1e-6, pos, _freq(128))
    want, _ = w4a4.qk_norm_rope(x, k, w, None, 1e-6, pos, _freq(128))
    clean = torch.ones((2, 3, 4), dtype=torch.bool, device="cuda")
    clean[0, 1, 2] = clean[1, 0, 0] = False
    assert torch.equal(got[clean], want[clean]) and torch.isnan(got[1, 0, 0]).all() and torch.isnan(got[0, 1, 2, 5])
    # a part that is not rotated does not meet the other half
    bad = x.clone()
    bad[0, 0, 0, 100] = float("inf")
    got, _ = w4a4.qk_norm_rope(bad, k, None, None, 0.0, pos, _freq(64))
    assert torch.isinf(got[0, 0, 0, 100]) and torch.isfinite(got[0, 0, 0, :100]).all() and torch.isfinite(got[0, 0, 0, 101:]).all()


# ------------------------------------------------------------------ into the cache
def _pool(gen, b, table_pages, kvh, d, dtype, spare=2):
    n = b * table_pages + spare
    cache = [torch.randn((n, kvh, PAGE, d), device="cuda", generator=gen).to(dtype) for _ in range(2)]
    table = torch.randperm(n, device="cuda", generator=gen)[: b * table_pages].to(torch.int32).view(b, table_pages)
    return cache, table


def _mirror(x, pool, table, lens, counts):
    pool = pool.clone()
    for b in range(x.size(0)):
        for i in range(min(max(counts[b], 0), x.size(1))):
            at = max(lens[b], 0) + i
            page = int(table[b, at // PAGE]) if at // PAGE < table.size(1) else -1
            if 0 <= page < pool.size(0):
                pool[page, :, at % PAGE] = x[b, i]
    return pool


CALLS = [(1, [0, 1, 63, 64], None), (1, [5, 0, 127, 100], [1, 0, 1, 1]), (3, [62, 63, 0, 10], None), (65, [0, 0, 30, 64], [65, 1, 40, 64]),
         (130, [0, 7, 64, 65], [130, 121, 0, 63]), (7, [250, 300, -4, 57], [7, 3, 9, -6])]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("h,kvh,d", [(8, 1, 256), (6, 2, 128), (3, 3, 64)])
@pytest.mark.parametrize("t,lens,counts", CALLS)
def test_append(cuda, t, lens, counts, h, kvh, d, dtype):
    """Plain and behind norm and rotation: the rows of the tokens, bit for bit, and nothing else."""
    gen = _gen(t + d)
    cache, table = _pool(gen, 4, 4, kvh, d, dtype)
    table[1, 1] = -1
    table[2, 0] = 10**6
    q, k, v = _heads(gen, 4, t, h, kvh, d, dtype)
    all_of = [t] * 4 if counts is None else counts
    c32 = None if counts is None else _i32(counts)
    want = [_mirror(x, c, table, lens, all_of) for x, c in zip((k, v), cache)]
    got = [c.clone() for c in cache]
    w4a4.kv_append(k, v, *got, table, _i32(lens), counts=c32)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])

    qw, kw = _weights(gen, d, dtype)
    pos = torch.randint(0, 900, (3, 4, t), device="cuda", generator=gen)
    axes = [j % 3 for j in range(d // 2)]
    qr, kr = w4a4.qk_norm_rope(q, k, qw, kw, 1e-6, pos, _freq(d), axes=axes)
    want = [_mirror(x, c, table, lens, all_of) for x, c in zip((kr, v), cache)]
    got = [c.clone() for c in cache]
    qo = w4a4.qk_norm_rope_append(q, k, v, qw, kw, 1e-6, pos, _freq(d), *got, table, _i32(lens), counts=c32, axes=axes)
    assert torch.equal(qo, qr) and torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_append_keeps_bits(cuda):
    """Infinities, NaN, zeros of either sign and the smallest numbers go through as they are."""
    bits = torch.arange(-32768, 32768, device="cuda", dtype=torch.int32).to(torch.int16).view(1, 1024, 1, 64)
    for dtype in TYPES:
        k = bits.view(dtype)
        cache = w4a4.kv_cache(17, 1, 64, dtype, "cuda")
        w4a4.kv_append(k, k.flip(1), *cache, torch.arange(16, device="cuda", dtype=torch.int32)[None], _i32([0]))
        assert torch.equal(cache[0][:16].view(torch.int16).view(-1), bits.view(-1))
        assert torch.equal(cache[1][:16].view(torch.int16).view(1, 1024, 1, 64), bits.flip(1)) and not cache[0][16].any()


def test_append_past_4_gib(cuda):
    n = 140000  # pages of 32 KB
    cache = w4a4.kv_cache(n, 1, 256, torch.float16, "cuda")
    k = torch.randn((1, 70, 1, 256), device="cuda", generator=_gen(8)).half()
    w4a4.kv_append(k, -k, *cache, _i32([[n - 1, 138000]]), _i32([0]))
    got = torch.cat([cache[0][n - 1, 0], cache[0][138000, 0, :6]])
    assert torch.equal(got, k[0, :, 0]) and torch.equal(cache[1][138000, 0, :6], -k[0, 64:, 0])
    assert not cache[0][138000, 0, 6:].any() and not cache[0][0].any()


def test_long_chunk(cuda):
    """Thousands of tokens: a wave takes all heads of one."""
    gen = _gen(9)
    q, k, v = _heads(gen, 2, 3001, 8, 1, 256, torch.bfloat16)
    qw, kw = _weights(gen, 256, torch.bfloat16)
    pos = torch.arange(3001, device="cuda", dtype=torch.int32)[None].expand(2, 3001)
    cache, table = _pool(gen, 2, 48, 1, 256, torch.bfloat16)
    qo = w4a4.qk_norm_rope_append(q, k, v, qw, kw, 1e-6, pos, _freq(256), *cache, table, _i32([0, 5]))
    _check(qo, q, qw, 1e-6, pos, _freq(256))
    for i, start in enumerate((0, 5)):
        rows = [c[table[i].long(), 0].reshape(-1, 256)[start:start + 3001] for c in cache]
        _check(rows[0][None, :, None].contiguous(), k[i:i + 1].contiguous(), kw, 1e-6, pos[:1], _freq(256))
        assert torch.equal(rows[1], v[i, :, 0])


def test_streams_and_graphs(cuda):
    """Two captured steps over their own caches, replayed in turn with moving inputs, equal the eager steps."""
    gen = _gen(10)
    qw, kw = _weights(gen, 128, torch.float16)
    freq, steps = _freq(128), []  # one tensor for both graphs, which keep reading it
    for _ in range(2):
        cache, table = _pool(gen, 3, 3, 2, 128, torch.float16)
        x = torch.zeros((3, 1, 8 * 128), device="cuda", dtype=torch.float16)
        lens, pos = _i32([0, 0, 0]), _i32([[0], [0], [0]])

        def call(x=x, cache=cache, table=table, lens=lens, pos=pos):
            h = x.view(3, 1, 8, 128)
            return w4a4.qk_norm_rope_append(h[:, :, :4], h[:, :, 4:6], h[:, :, 6:], qw, kw, 1e-6, pos, freq, *cache, table, lens)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        steps.append((graph, out, x, cache, table, lens, pos, call))
    for i in range(20):
        for graph, out, x, cache, table, lens, pos, call in steps:
            x.copy_(torch.randn(x.shape, device="cuda", generator=gen))
            lens.copy_(_i32([i, 100 + i, 63]))
            pos.copy_(_i32([[i], [7 * i], [3]]))
            keep = [c.clone() for c in cache]
            graph.replay()
            after = [c.clone() for c in cache]
            got = out.clone()
            for c, was in zip(cache, keep):
                c.copy_(was)
            want = call()
            torch.cuda.synchronize()
            assert torch.equal(got, want) and all(torch.equal(a, c) for a, c in zip(after, cache))


def test_refusals(cuda):
    q = torch.zeros((2, 3, 4, 64), dtype=torch.float16, device="cuda")
    k, pos, freq = q[:, :, :2], torch.zeros((2, 3), dtype=torch.int32, device="cuda"), _freq(64)
    w = q[0, 0, 0]

    def call(q=q, k=k, qw=None, kw=None, eps=1e-6, pos=pos, freq=freq, **kw2):
        return w4a4.qk_norm_rope(q, k, qw, kw, eps, pos, freq, **kw2)

    for kw, text in [
        (dict(q=q.float()), "of one type"), (dict(k=k.bfloat16()), "of one type"), (dict(k=k[:, :2]), "expects q"), (dict(q=q[0]), "expects q"),
        (dict(k=k[..., :32]), "expects q"), (dict(k=k.cpu()), "one device"), (dict(q=q[..., :40], k=k[..., :40]), "multiple of 16"),
        (dict(qw=w.float()), "q_weight"), (dict(kw=w[:32]), "k_weight"), (dict(freq=freq.double()), "inv_freq"), (dict(freq=freq.cpu()), "inv_freq"),
        (dict(freq=_freq(80)), "rotated dimensions"), (dict(freq=freq[:4]), "rotated dimensions"), (dict(pos=pos.float()), "positions"),
        (dict(pos=pos[:1]), "positions"), (dict(pos=pos[None].expand(5, 2, 3)), "positions"), (dict(pos=pos.cpu()), "positions"),
        (dict(pos=pos[None].expand(3, 2, 3)), "need `axes`"), (dict(axes=[0] * 31), "axes must name"), (dict(axes=[1] * 32), r"in \[0, 1\)"),
        (dict(pos=pos[None].expand(3, 2, 3), axes=[3] * 32), r"in \[0, 3\)"), (dict(eps=float("nan")), "eps"), (dict(eps=-1.0), "eps"),
        (dict(q=q[:, :, :0]), "heads"),
    ]:
        with pytest.raises(RuntimeError, match=text):
            call(**kw)
    assert call(q=q[:0], k=k[:0], pos=pos[:0])[0].shape == (0, 3, 4, 64) and call(q=q[:, :0], k=k[:, :0], pos=pos[:, :0])[1].numel() == 0
    cache = w4a4.kv_cache(2, 2, 64, torch.float16, "cuda")
    table, lens = _i32([[0], [1]]), _i32([0, 0])

    def append(cache=cache, v=k, table=table, lens=lens, **kw):
        return w4a4.qk_norm_rope_append(q, k, v, None, None, 0.0, pos, freq, *cache, table, lens, **kw)

    for kw, text in [(dict(v=k.bfloat16()), "v must be"), (dict(v=k[:, :1]), "v must be"), (dict(cache=[c.bfloat16() for c in cache]), "k_cache"),
                     (dict(cache=[cache[0], cache[1][:1]]), "v_cache"), (dict(table=table.long()), "block_table"), (dict(lens=lens[:1]), "lens"),
                     (dict(cache=[c.cpu() for c in cache]), "must be on"), (dict(counts=lens.long()), "counts"),
                     (dict(cache=[c.transpose(0, 1).contiguous().transpose(0, 1) for c in cache]), "contiguous")]:
        with pytest.raises(RuntimeError, match=text):
            append(**kw)
    leaf = q.clone().requires_grad_()
    with pytest.raises((RuntimeError, NotImplementedError)):
        w4a4.qk_norm_rope(leaf, k, None, None, 0.0, pos, freq)[0].sum().backward()


def test_dispatched_route(cuda):
    gen = _gen(11)
    q, k, v = _heads(gen, 2, 3, 4, 2, 64, torch.float16)
    qw, kw = _weights(gen, 64, torch.float16)
    pos, freq, axes = _i32([[[1, 2, 3], [4, 5, 6]]] * 2), _freq(64), [j % 2 for j in range(32)]
    cache, table = _pool(gen, 2, 2, 2, 64, torch.float16)
    other = [c.clone() for c in cache]

    def step(q, k, v, kc, vc):
        a, b = w4a4.qk_norm_rope(q, k, qw, kw, 1e-6, pos, freq, axes=axes)
        w4a4.kv_append(b, v, kc, vc, table, _i32([3, 70]))
        return a, w4a4.qk_norm_rope_append(q, k, v, qw, kw, 1e-6, pos, freq, kc, vc, table, _i32([10, 80]), axes=axes)

    want = step(q, k, v, *cache)
    got = torch.compile(step, fullgraph=True, backend="eager")(q, k, v, *other)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and all(torch.equal(a, b) for a, b in zip(cache, other))

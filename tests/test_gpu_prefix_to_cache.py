"""The framework's own way to the 16-bit cache: INT4 products with adapters, ``prefix_attention``, its key states and
values into the cache, and the tokens behind the prefix over it."""

from __future__ import annotations

import pytest
import torch
from test_gpu_attention import REL_L2, _padding_causal_mask, _rotary
from test_gpu_kv import _gen, _i32, _pool, _reference
from test_gpu_lora import _ref

from pi05_fast import w4a4
from pi05_fast.w4a4 import extension as ext

pytestmark = pytest.mark.gpu
WIDTH, D = 512, 256


@pytest.mark.parametrize("h,kvh,s", [(8, 1, 72), (4, 2, 130)])
def test_prefix_attention_to_the_cache(cuda, h, kvh, s):
    gen = _gen(s)
    b, t, lengths = 3, 5, [s, s - 9, 65]
    x = torch.randn((b, s, WIDTH), device="cuda", generator=gen).half()
    ids = _i32([1, -1, 0])
    heads = []
    for n in (h, kvh, kvh):
        w = w4a4.pack_linear_weight(torch.randn((n * D, WIDTH), generator=torch.Generator().manual_seed(n)) * WIDTH**-0.5).cuda()
        y = ext.int4_gemm(x, w)
        a, bb = ((torch.randn(size, device="cuda", generator=gen) * 0.1).half() for size in ((2, 16, WIDTH), (2, n * D, 16)))
        got = w4a4.lora_add(y, x, a, bb, ids)
        want, tol = _ref(y.flatten(0, 1), x.flatten(0, 1), a, bb, ids.repeat_interleave(s), None, [n * D])
        assert ((got.flatten(0, 1).double() - want).abs() <= tol).all()
        heads.append(got)
    q, k, v = heads
    cos, sin = _rotary(b, s, cuda)
    out, keys = ext.prefix_attention(q, k, v, cos, sin, _padding_causal_mask(b, s, lengths, cuda), D**-0.5, h, kvh)

    cache, table = _pool(gen, b, 4, kvh, D, torch.float16)
    was, lens = [c.clone() for c in cache], _i32(lengths)
    w4a4.kv_append(keys.transpose(1, 2), v.unflatten(-1, (kvh, D)), *cache, table, torch.zeros_like(lens), counts=lens)
    for i, n in enumerate(lengths):
        for c, old, new in zip(cache, was, (keys[i], v[i].unflatten(-1, (kvh, D)).transpose(0, 1))):
            rows, before = (pool[table[i].long()].transpose(0, 1).flatten(1, 2) for pool in (c, old))  # [KVH, tokens, D]
            assert torch.equal(rows[:, :n], new[:, :n]) and torch.equal(rows[:, n:], before[:, n:])

    # the prefix's own queries over the cache are what prefix_attention gave
    freq = (10000.0 ** (-torch.arange(D // 2, device="cuda", dtype=torch.float64) / (D // 2))).float()
    pos = torch.arange(s, device="cuda")[None].expand(b, s)
    turned, again = w4a4.qk_norm_rope(q.unflatten(-1, (h, D)), k.unflatten(-1, (kvh, D)), None, None, 0.0, pos, freq)
    # key states in units of half a step of the largest k: sines and products rounded, 2 of each of two terms, their sum 1.42
    # times as large rounded, and the one rounding of the other side
    assert ((again.transpose(1, 2).float() - keys.float()).abs() <= 7 * 2.0**-11 * k.float().abs().amax()).all()
    got = w4a4.kv_attention(turned, *cache, table, lens, D**-0.5, q_lens=lens).flatten(2)
    for i, n in enumerate(lengths):
        one, two = got[i, :n].double(), out[i, :n].double()
        # prefix_attention is held to REL_L2 of the fp32 result, kv_attention rounds once
        assert (one - two).norm() <= (REL_L2 + 2.0**-11) * two.norm()

    # tokens behind the prefix, which see it and each other
    qn, kn, vn = (torch.randn((b, t, n, D), device="cuda", generator=gen).half() for n in (h, kvh, kvh))
    pos = lens[:, None] + torch.arange(t, device="cuda")
    qn = w4a4.qk_norm_rope_append(qn, kn, vn, None, None, 0.0, pos, freq, *cache, table, lens)
    act = w4a4.kv_attention(qn, *cache, table, lens + t, D**-0.5, causal=False)
    want, _, tol, _ = _reference(qn, cache, table, [n + t for n in lengths], D**-0.5, False, None)
    assert ((act.double() - want).abs() <= tol).all()

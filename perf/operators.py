"""Performance cases of the 8-bit operators: int8 rows, int8 products and the int8 KV cache.

One pass is one call of an operator as a program makes it.  With ``own`` the calls go to the
package (``pi05_fast.w4a4``); without it they are computed from elementary torch operations in
32 bits, rounded once at the end.

* ``add_norm``, ``norm``, ``quantize``   rows to 8-bit codes with a scale each: behind a residual
                add and an RMSNorm, behind an RMSNorm, or as they are;
* ``gemm``      int8 codes x int8 weights with token and channel scales, with a bias, a residual
                or neither;
* ``append``    new keys and values into an 8-bit cache of 64-token pages, one scale for each page
                and KV head (keys and values have their own);
* ``attend``    attention of the last tokens of each sequence over such a cache.

Codes are returned as the values they stand for (code * scale), in the inputs' type.

Sizes are PaliGemma-2B's (hidden 2048, intermediate 16384, 8 query heads and 1 KV head of 256,
776-token prefixes, batches up to 8 of them, 8192 positions), the 50 action tokens that attend
to a prefix, and generic widths and head layouts.  Activations are N(0, 1) with 1% of the
channels 20 times larger; cached keys and values are N(0, 1) with a level of its own for each
page, quantized by page; slots behind a sequence's last token hold what an earlier sequence left.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

_PKG = str(Path(__file__).resolve().parents[1] / "pi05-pytorch-fast_amd")
if _PKG not in sys.path:
    sys.path.insert(0, _PKG)

PAGE = 64
EPS = 1e-6
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # a decoded token's residual stream into the codes of its next projection: latency
        {"name": "add_norm_1x2048", "op": "add_norm", "rows": 1, "k": 2048, "dtype": "fp16"},
        # the same for a batch of eight 776-token prefixes: bandwidth
        {"name": "add_norm_6208x2048", "op": "add_norm", "rows": 6208, "k": 2048, "dtype": "bf16"},
        # a decoded token through the joined QKV projection
        {"name": "gemm_1_qkv", "op": "gemm", "rows": 1, "k": 2048, "n": 2560, "extra": "none", "dtype": "fp16"},
        # a batch of decoded tokens through the down projection, with the residual
        {"name": "gemm_64_down", "op": "gemm", "rows": 64, "k": 16384, "n": 2048, "extra": "residual", "dtype": "fp16"},
        # one 776-token prefix through the joined QKV projection
        {"name": "gemm_776_qkv", "op": "gemm", "rows": 776, "k": 2048, "n": 2560, "extra": "none", "dtype": "fp16"},
        # eight prefixes through one of the MLP's wide projections, as a layer with a bias
        {"name": "gemm_6208_wide", "op": "gemm", "rows": 6208, "k": 2048, "n": 16384, "extra": "bias", "dtype": "bf16"},
        # the keys and values of one decoded token for each of 16 requests
        {"name": "append_16x1", "op": "append", "batch": 16, "tokens": 1, "ctx": 776, "kv_heads": 1, "d": 256, "dtype": "fp16"},
        # eight whole prefixes into an empty cache
        {"name": "append_8x776", "op": "append", "batch": 8, "tokens": 776, "ctx": 0, "kv_heads": 1, "d": 256, "dtype": "fp16"},
        # one decoded token over one prefix: latency
        {"name": "attend_1x1_776", "op": "attend", "batch": 1, "tokens": 1, "ctx": 776, "heads": 8, "kv_heads": 1, "d": 256,
         "causal": True, "dtype": "fp16"},
        # a decode step of 64 requests with up to 8192 tokens: the cache's bandwidth
        {"name": "attend_64x1_8192", "op": "attend", "batch": 64, "tokens": 1, "ctx": 8192, "heads": 8, "kv_heads": 1, "d": 256,
         "causal": True, "dtype": "fp16"},
        # the action tokens of eight requests over their prefixes and themselves, in both directions
        {"name": "attend_8x50_826", "op": "attend", "batch": 8, "tokens": 50, "ctx": 826, "heads": 8, "kv_heads": 1, "d": 256,
         "causal": False, "dtype": "bf16"},
        # a prompt's next 776 tokens behind a long cached context, two requests
        {"name": "attend_2x776_4096", "op": "attend", "batch": 2, "tokens": 776, "ctx": 4096, "heads": 8, "kv_heads": 1, "d": 256,
         "causal": True, "dtype": "fp16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_MOST_MACS = 6208 * 2048 * 16384
_HEADS = ((8, 1, 256), (8, 2, 256), (16, 4, 128), (8, 8, 64), (6, 2, 128), (32, 8, 64))


def draw(rng):
    op = rng.choice(["add_norm", "norm", "quantize", "gemm", "gemm", "gemm", "append", "append", "attend", "attend", "attend"])
    dtype = rng.choice(["fp16", "bf16"])
    if op in ("add_norm", "norm", "quantize"):
        return {"op": op, "rows": _log(rng, 1, 6208), "k": rng.choice([8 * _log(rng, 16, 1024), 1024, 2048, 4096, 16384]),
                "dtype": dtype}
    if op == "gemm":
        rows, k = _log(rng, 1, 6208), rng.choice([16 * _log(rng, 8, 1024), 1024, 2048, 4096, 16384])
        n = rng.choice([_log(rng, 8, 16384), 16 * _log(rng, 8, 1024)])
        n = max(8, min(n, _MOST_MACS // (rows * k)))
        return {"op": op, "rows": rows, "k": k, "n": n, "extra": rng.choice(["none", "bias", "residual"]), "dtype": dtype}
    heads, kv_heads, d = rng.choice(_HEADS)
    if op == "append":
        batch = _log(rng, 1, 32)
        tokens = rng.choice([1, _log(rng, 1, 776)])
        tokens = max(1, min(tokens, 8 * 776 * 512 // (batch * 2 * kv_heads * d)))
        return {"op": op, "batch": batch, "tokens": tokens, "ctx": rng.randint(0, 776), "kv_heads": kv_heads, "d": d, "dtype": dtype}
    batch = _log(rng, 1, 64)
    ctx = _log(rng, 1, 8192)
    tokens = min(ctx, rng.choice([1, 1, _log(rng, 2, 776)]))
    # no more cached bytes than 64 x 8192 tokens of one head of 256, no more scores than two 776-token chunks over 4096
    batch = max(1, min(batch, 64 * 8192 * 256 // (ctx * kv_heads * d), 2 * 776 * 4096 * 8 // (tokens * ctx * heads)))
    while tokens > 1 and batch * tokens * ctx * heads * d > 2 * 776 * 4096 * 8 * 256:
        tokens //= 2
    return {"op": op, "batch": batch, "tokens": tokens, "ctx": ctx, "heads": heads, "kv_heads": kv_heads, "d": d,
            "causal": rng.random() < 0.7, "dtype": dtype}


# ------------------------------------------------------------------ inputs, from the seed
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(0x8B17 + int(seed))


def _activations(gen, *shape):
    x = torch.randn(shape, device="cuda", generator=gen)
    cols = torch.randperm(shape[-1], device="cuda", generator=gen)[: max(1, shape[-1] // 100)]
    x[..., cols] *= 20.0
    return x


def _codes(x):
    """Rows of x as int8 codes with a scale each."""
    s = x.abs().amax(dim=-1) / 127.0 + 1e-12
    return torch.round(x / s[..., None]).clamp_(-127, 127).to(torch.int8), s


def _cache(gen, case, pages_each, lens):
    """A pool of pages in a random order: (k_cache [P, KVH, 64, D], v_cache [P, KVH, D, 64], k_scale, v_scale [P, KVH],
    block_table [B, pages_each])."""
    b, kvh, d = case["batch"], case["kv_heads"], case["d"]
    n = b * pages_each
    table = torch.randperm(n, device="cuda", generator=gen).to(torch.int32).view(b, pages_each)

    def side():
        codes = torch.empty((n, kvh, PAGE, d), dtype=torch.int8, device="cuda")
        scale = torch.empty((n, kvh), dtype=torch.float32, device="cuda")
        for p in range(0, n, 512):
            x = torch.randn((min(512, n - p), kvh, PAGE, d), device="cuda", generator=gen)
            x *= torch.rand((x.size(0), kvh, 1, 1), device="cuda", generator=gen) * 0.8 + 0.6
            c, s = _codes(x.flatten(2))
            codes[p:p + 512], scale[p:p + 512] = c.view(x.shape), s
        return codes, scale

    kc, ks = side()
    vc, vs = side()
    return kc, vc.transpose(2, 3).contiguous(), ks, vs, table


def _lens(gen, batch, lo, hi):
    return torch.randint(lo, hi + 1, (batch,), device="cuda", generator=gen).to(torch.int32)


@torch.no_grad()
def prepare(case, seed):
    gen, op = _gen(seed), case["op"]
    t = DTYPES[case["dtype"]]
    s = {"op": op, "t": t}
    if op in ("add_norm", "norm", "quantize"):
        s["x"] = _activations(gen, case["rows"], case["k"]).to(t)
        if op == "add_norm":
            s["res"] = (_activations(gen, case["rows"], case["k"]) * 2.0).to(t)
        if op != "quantize":
            s["w"] = (torch.randn((case["k"],), device="cuda", generator=gen) * 0.05).to(t)
        return s
    if op == "gemm":
        m, k, n = case["rows"], case["k"], case["n"]
        s["q"], s["sq"] = _codes(_activations(gen, m, k))
        s["w"], s["sw"] = _codes(torch.randn((n, k), device="cuda", generator=gen) * 0.02)
        s["bias"] = (torch.randn((n,), device="cuda", generator=gen) * 0.1).to(t) if case["extra"] == "bias" else None
        s["res"] = _activations(gen, m, n).to(t) if case["extra"] == "residual" else None
        return s
    b, tokens, kvh, d = case["batch"], case["tokens"], case["kv_heads"], case["d"]
    if op == "append":
        s["lens"] = _lens(gen, b, 3 * case["ctx"] // 4, case["ctx"])
        s["kc"], s["vc"], s["ks"], s["vs"], s["table"] = _cache(gen, case, case["ctx"] // PAGE + (tokens + 62) // PAGE + 2, s["lens"])
        # keys are usually of the pages' own level; now and then a page's scale has to grow
        s["k"], s["v"] = ((torch.randn((b, tokens, kvh, d), device="cuda", generator=gen)
                           * (torch.rand((b, tokens, 1, 1), device="cuda", generator=gen) * 0.8 + 0.6)).to(t) for _ in range(2))
        s["counts"] = _lens(gen, b, max(1, tokens - tokens // 4), tokens)
        return s
    lo = max(tokens, case["ctx"] - (case["ctx"] // 2 if b > 1 else 0))
    s["lens"] = _lens(gen, b, lo, case["ctx"])
    s["kc"], s["vc"], s["ks"], s["vs"], s["table"] = _cache(gen, case, (case["ctx"] + PAGE - 1) // PAGE, s["lens"])
    s["q"] = (torch.randn((b, tokens, case["heads"], d), device="cuda", generator=gen) * 1.5).to(t)
    s["causal"], s["scaling"] = case["causal"], d**-0.5
    return s


# ------------------------------------------------------------------ the calls
def _values(codes, scale, t):
    """Codes as the values they stand for, in one launch."""
    return torch.mul(codes, scale, out=torch.empty(codes.shape, dtype=t, device=codes.device))


@torch.no_grad()
def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    from pi05_fast.w4a4 import int8 as i8
    from pi05_fast.w4a4 import kv_int8 as kv

    op = s["op"]
    if op == "add_norm":
        q, sq, h = i8.add_rms_norm_int8(s["x"], s["res"], s["w"], EPS)
        return _values(q, sq[:, None], s["t"]), h
    if op == "norm":
        q, sq = i8.rms_norm_int8(s["x"], s["w"], EPS)
        return _values(q, sq[:, None], s["t"])
    if op == "quantize":
        q, sq = i8.quantize_int8(s["x"])
        return _values(q, sq[:, None], s["t"])
    if op == "gemm":
        return i8.int8_gemm(s["q"], s["sq"], s["w"], s["sw"], bias=s["bias"], residual=s["res"], out_dtype=s["t"])
    if op == "append":
        kv.int8_kv_append(s["k"], s["v"], s["kc"], s["vc"], s["ks"], s["vs"], s["table"], s["lens"], counts=s["counts"])
        return _values(s["kc"], s["ks"][..., None, None], s["t"]), _values(s["vc"], s["vs"][..., None, None], s["t"])
    return kv.int8_kv_attention(s["q"], s["kc"], s["vc"], s["ks"], s["vs"], s["table"], s["lens"], s["scaling"],
                                causal=s["causal"])


def _rows_plain(y, t):
    step = y.abs().amax(dim=-1, keepdim=True) / 127.0 + 1e-12
    return (torch.round(y * (1.0 / step)).clamp_(-127, 127) * step).to(t)


def _append_side(x, codes, scale, table, lens, counts):
    """The touched pages' new codes [B, n, KVH, 64, D] and scales [B, n, KVH] of one side, and those pages' places in the
    pool.  ``codes`` is the pool as [P, KVH, 64, D]."""
    b, tokens, kvh, d = x.shape
    n = (tokens + 62) // PAGE + 1
    slot = (lens // PAGE)[:, None] + torch.arange(n, device=x.device)[None]
    phys = table.long().gather(1, slot.long())
    # token of each place in the touched pages: -1 and below: there already, counts and above: empty
    tok = slot[..., None] * PAGE + torch.arange(PAGE, device=x.device) - lens[:, None, None]
    new = (tok >= 0) & (tok < counts[:, None, None])
    rows = x.float()[torch.arange(b, device=x.device)[:, None, None], tok.clamp(0, tokens - 1).long()]  # [B, n, 64, KVH, D]
    rows = torch.where(new[..., None, None], rows, torch.zeros((), device=x.device)).transpose(2, 3)
    there = (slot * PAGE < lens[:, None])[..., None]
    s0 = torch.where(there, scale[phys], torch.zeros((), device=x.device))
    top = rows.abs().amax(dim=(3, 4))
    touched = new.any(-1)[..., None]
    s1 = torch.where(touched, torch.maximum(s0, top / torch.full_like(top, 127.0) + 1e-12), scale[phys])
    old = codes[phys].float()
    ratio = torch.where(touched & (s1 > s0), s0 / s1, torch.ones((), device=x.device))
    old = torch.round(old * ratio[..., None, None])
    fresh = torch.round(rows * (1.0 / s1)[..., None, None]).clamp_(-127, 127)
    return torch.where(new[:, :, None, :, None], fresh, old).to(torch.int8), s1, phys


def _pages(codes, scale, table):
    """A cache side as values [B, KVH, tokens, D] in the scales' type."""
    b, p = table.shape
    x = codes[table.long()].to(scale.dtype) * scale[table.long()][..., None, None]  # [B, pages, KVH, 64, D]
    return x.transpose(1, 2).reshape(b, x.size(2), p * PAGE, x.size(-1))


def _attend(q, k, v, lens, scaling, causal):
    """q [B, T, H, D] over k, v [B, KVH, L, D], in their type."""
    b, t, h, d = q.shape
    kvh = k.size(1)
    rows = q.to(k.dtype).view(b, t, kvh, h // kvh, d).permute(0, 2, 1, 3, 4).reshape(b, kvh, t * (h // kvh), d)
    score = torch.matmul(rows, k.transpose(2, 3).contiguous()) * scaling
    tok = torch.arange(t, device=q.device).repeat_interleave(h // kvh)
    seen = lens[:, None] - t + tok[None] + 1 if causal else lens[:, None].expand(b, tok.numel())
    hidden = torch.arange(k.size(2), device=q.device)[None, None] >= seen[..., None]
    score = score.masked_fill_(hidden[:, None], float("-inf"))
    top = score.amax(dim=-1, keepdim=True)
    p = torch.exp(score - torch.where(torch.isinf(top), torch.zeros((), device=q.device, dtype=top.dtype), top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / torch.where(total == 0, torch.ones((), device=q.device, dtype=total.dtype), total)
    return out.view(b, kvh, t, h // kvh, d).permute(0, 2, 1, 3, 4).reshape(b, t, h, d)


def _run_plain(s):
    op, t = s["op"], s["t"]
    if op in ("add_norm", "norm", "quantize"):
        x = s["x"].float()
        if op == "quantize":
            return _rows_plain(x, t)
        h = (x + s["res"].float()).to(t) if op == "add_norm" else None
        f = h.float() if op == "add_norm" else x
        y = f * (1.0 / torch.sqrt(f.square().mean(dim=-1, keepdim=True) + EPS)) * (1.0 + s["w"].float())
        return (_rows_plain(y, t), h) if op == "add_norm" else _rows_plain(y, t)
    if op == "gemm":
        y = torch.matmul(s["q"].float(), s["w"].float().t()) * s["sq"][:, None] * s["sw"]
        if s["bias"] is not None:
            y = y + s["bias"].float()
        if s["res"] is not None:
            y = y + s["res"].float()
        return y.to(t)
    if op == "append":
        for x, pool, scale, turn in ((s["k"], s["kc"], s["ks"], False), (s["v"], s["vc"], s["vs"], True)):
            codes, s1, phys = _append_side(x, pool.transpose(2, 3) if turn else pool, scale, s["table"], s["lens"], s["counts"])
            pool[phys] = codes.transpose(3, 4) if turn else codes
            scale[phys] = s1
        return _values(s["kc"], s["ks"][..., None, None], t), _values(s["vc"], s["vs"][..., None, None], t)
    k = _pages(s["kc"], s["ks"], s["table"])
    v = _pages(s["vc"].transpose(2, 3), s["vs"], s["table"])
    return _attend(s["q"], k, v, s["lens"], s["scaling"], s["causal"]).to(t)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    op = case["op"]
    if op in ("add_norm", "norm", "quantize"):
        m, k = case["rows"], case["k"]
        # the rows (and the residual) in, the codes and scales (and the new stream) out
        return {"bytes": float(m * k * (7 if op == "add_norm" else 3) + 4 * m + (0 if op == "quantize" else 2 * k)),
                "flops": float(m * k * (4 if op == "quantize" else 8))}
    if op == "gemm":
        m, k, n = case["rows"], case["k"], case["n"]
        extra = {"none": 0, "bias": 2 * n, "residual": 2 * m * n}[case["extra"]]
        return {"bytes": float(m * k + n * k + 2 * m * n + 4 * (m + n) + extra), "flops": 2.0 * m * k * n}
    b, t, kvh, d = case["batch"], case["tokens"], case["kv_heads"], case["d"]
    if op == "append":
        # keys and values in, their codes out, and a scale for each page
        rows = 2.0 * b * t * kvh * d
        return {"bytes": 3.0 * rows + 8.0 * b * kvh * (t + 63) // 64, "flops": 4.0 * rows}
    length = case["ctx"] * (0.75 if b > 1 else 1.0)  # sequences of a batch are half to all of ctx
    return {"bytes": 2.0 * b * kvh * d * length + 4.0 * b * t * case["heads"] * d, "flops": 4.0 * b * case["heads"] * t * length * d}


# ------------------------------------------------------------------ 64-bit results
@torch.no_grad()
def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    f64 = torch.float64
    if op in ("add_norm", "norm", "quantize"):
        y, h = s["x"].to(f64), None
        if op == "add_norm":
            h = y = (y + s["res"].to(f64)).to(s["t"]).to(f64)
        if op != "quantize":
            y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / y.size(-1) + EPS) * (s["w"].to(f64) + 1)
        step = torch.linalg.vector_norm(y, ord=float("inf"), dim=-1, keepdim=True) / 127 + 1e-12
        y = torch.clamp(torch.round(y / step), -127, 127) * step
        return (y, h) if op == "add_norm" else y
    if op == "gemm":
        # 53 bits hold the integer sums exactly
        y = s["q"].to(f64) @ s["w"].to(f64).t().contiguous()
        y = s["sq"].to(f64)[:, None] * (y * s["sw"].to(f64)[None])
        y += 0 if s["bias"] is None else s["bias"].to(f64)
        return y + (0 if s["res"] is None else s["res"].to(f64))
    if op == "append":
        out = []
        for x, pool, scale, turn in ((s["k"], s["kc"], s["ks"], False), (s["v"], s["vc"], s["vs"], True)):
            codes = (pool.transpose(2, 3) if turn else pool).to(f64).clone()
            scale = scale.to(f64).clone()
            for i, (have, count) in enumerate(zip(s["lens"].tolist(), s["counts"].tolist())):
                at = 0
                while at < count:
                    page = int(s["table"][i, (have + at) // PAGE])
                    o = (have + at) % PAGE
                    m = min(PAGE - o, count - at)
                    rows = x[i, at:at + m].to(f64).transpose(0, 1)  # [KVH, m, D]
                    need = rows.abs().flatten(1).amax(1) / 127 + 1e-12
                    grown = torch.maximum(need, scale[page]) if o else need
                    # a new page starts empty; in one that has tokens their codes follow its scale
                    codes[page] = torch.round(codes[page] * (scale[page] / grown)[:, None, None]) if o else 0.0
                    codes[page, :, o:o + m] = torch.clamp(torch.round(rows / grown[:, None, None]), -127, 127)
                    scale[page] = grown
                    at += m
            y = codes * scale[:, :, None, None]
            out.append(y.transpose(2, 3).contiguous() if turn else y)
        return tuple(out)
    out = torch.empty(s["q"].shape, dtype=f64, device="cuda")
    group = case["heads"] // case["kv_heads"]
    for i, length in enumerate(s["lens"].tolist()):
        ids = s["table"][i, : (length + PAGE - 1) // PAGE].long()
        for g in range(case["kv_heads"]):
            k = (s["kc"][ids, g].to(f64) * s["ks"][ids, g].to(f64)[:, None, None]).reshape(-1, case["d"])[:length]
            v = (s["vc"][ids, g].to(f64) * s["vs"][ids, g].to(f64)[:, None, None]).transpose(1, 2).reshape(-1, case["d"])[:length]
            for h in range(g * group, (g + 1) * group):
                z = (s["q"][i, :, h].to(f64).contiguous() @ k.t().contiguous()) * s["scaling"]
                if s["causal"]:
                    last = length - case["tokens"] + torch.arange(case["tokens"], device="cuda")
                    z = z.masked_fill(torch.arange(length, device="cuda")[None] > last[:, None], float("-inf"))
                out[i, :, h] = torch.softmax(z, dim=-1) @ v
    return out

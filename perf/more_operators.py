"""Performance cases of the operators around a 16-bit KV cache: head norms and rotary positions, the
cache's append and attention, and the low-rank adapters of many requests.

One pass is one call of an operator as a program makes it.  With ``own`` the calls go to the
package (``pi05_fast.w4a4``); without it they are computed from elementary torch operations in
32 bits (angles in 64), rounded once at the end.

* ``rope``         an RMSNorm of each query and key head and the rotation by position, in one pass, with
                   one position a token or several (time, height, width);
* ``rope_append``  the same, with the keys and values written into a paged 16-bit cache;
* ``append``       keys and values as they are into that cache;
* ``attend``       attention of the last tokens of each sequence over that cache;
* ``lora``         y + scale * (x A^T) B^T beside a shared projection, A, B and scale those of each
                   row's request.

Sizes are PaliGemma-2B's (hidden 2048, intermediate 16384, 8 query heads and 1 KV head of 256,
776-token prefixes, batches up to 8 of them, 8192 positions), the 50 action tokens that attend
to a prefix, and generic widths, ranks and head layouts.  Activations are N(0, 1) with 1% of the
channels 20 times larger; cached keys and values are N(0, 1); slots behind a sequence's last token
hold what an earlier sequence left.
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
THETA = 10000.0
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one decoded token's joined QKV output: latency
        {"name": "rope_1x1", "op": "rope", "batch": 1, "tokens": 1, "ctx": 776, "heads": 8, "kv_heads": 1, "d": 256, "rot": 256,
         "axes": 1, "mixed": False, "interleaved": False, "norm": True, "dtype": "fp16"},
        # a batch of images and text with positions of three axes, wide head layout: bandwidth
        {"name": "rope_4x1536_axes", "op": "rope", "batch": 4, "tokens": 1536, "ctx": 4096, "heads": 32, "kv_heads": 8, "d": 128,
         "rot": 128, "axes": 3, "mixed": False, "interleaved": False, "norm": True, "dtype": "bf16"},
        # the queries, keys and values of one decoded token for each of 64 requests
        {"name": "rope_append_64x1", "op": "rope_append", "batch": 64, "tokens": 1, "ctx": 776, "heads": 8, "kv_heads": 1, "d": 256,
         "rot": 256, "axes": 1, "mixed": False, "interleaved": False, "norm": True, "dtype": "bf16"},
        # eight whole prefixes on their way into an empty cache
        {"name": "rope_append_8x776", "op": "rope_append", "batch": 8, "tokens": 776, "ctx": 0, "heads": 8, "kv_heads": 1, "d": 256,
         "rot": 256, "axes": 1, "mixed": False, "interleaved": False, "norm": True, "dtype": "fp16"},
        # keys that are rotated already: one decoded token for each of 16 requests
        {"name": "append_16x1", "op": "append", "batch": 16, "tokens": 1, "ctx": 776, "kv_heads": 1, "d": 256, "dtype": "fp16"},
        # the key states and values of eight prefixes, as the prefix attention returns them
        {"name": "append_8x776", "op": "append", "batch": 8, "tokens": 776, "ctx": 0, "kv_heads": 1, "d": 256, "dtype": "fp16"},
        # one decoded token over one prefix: latency
        {"name": "attend_1x1_776", "op": "attend", "batch": 1, "tokens": 1, "ctx": 776, "heads": 8, "kv_heads": 1, "d": 256,
         "causal": True, "dtype": "fp16"},
        # a decode step of 64 requests with up to 8192 tokens: the cache's bandwidth
        {"name": "attend_64x1_8192", "op": "attend", "batch": 64, "tokens": 1, "ctx": 8192, "heads": 8, "kv_heads": 1, "d": 256,
         "causal": True, "dtype": "bf16"},
        # the action tokens of eight requests over their prefixes and themselves, in both directions
        {"name": "attend_8x50_826", "op": "attend", "batch": 8, "tokens": 50, "ctx": 826, "heads": 8, "kv_heads": 1, "d": 256,
         "causal": False, "dtype": "bf16"},
        # one decoded token with an adapter on each part of the joined QKV projection: latency
        {"name": "lora_1_qkv", "op": "lora", "batch": 1, "tokens": 1, "k": 2048, "n": 2560, "rank": 16, "slices": 3, "adapters": 8,
         "dtype": "fp16"},
        # a decode step of 64 requests with an adapter each on the output projection
        {"name": "lora_64_o", "op": "lora", "batch": 64, "tokens": 1, "k": 2048, "n": 2048, "rank": 16, "slices": 1, "adapters": 64,
         "dtype": "bf16"},
        # eight prefixes of five adapters through the joined gate and up projection
        {"name": "lora_8x776_gate_up", "op": "lora", "batch": 8, "tokens": 776, "k": 2048, "n": 32768, "rank": 32, "slices": 2,
         "adapters": 5, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_HEADS = ((8, 1, 256), (8, 2, 256), (16, 4, 128), (8, 8, 64), (6, 2, 128), (32, 8, 64), (32, 8, 128))
# head widths that only the rotation takes
_OTHER_HEADS = ((5, 5, 80), (12, 3, 96), (4, 1, 512), (7, 7, 112))
_MOST_ROPE = 4 * 1536 * (32 + 8) * 128
_MOST_ROWS = 8 * 776 * (2048 + 2 * 32768) * 7 // 8
_MOST_PRODUCTS = 8 * 776 * 32 * (2 * 2048 + 32768) * 7 // 8
_MOST_WEIGHTS = 1 << 25


def draw(rng):
    op = rng.choice(["rope", "rope", "rope_append", "rope_append", "append", "attend", "attend", "attend", "lora", "lora", "lora"])
    dtype = rng.choice(["fp16", "bf16"])
    if op == "lora":
        batch = _log(rng, 1, 256)
        tokens = rng.choice([1, 1, _log(rng, 1, 776)])
        k = rng.choice([8 * _log(rng, 16, 2048), 1024, 2048, 4096, 16384])
        slices = rng.choice([1, 1, 2, 3])
        n = rng.choice([2560, 2048, 16384, 16 * _log(rng, 8, 1024), _log(rng, 64, 16384)]) if slices == 1 else 48 * _log(rng, 8, 512)
        rank, adapters = rng.choice([8, 16, 32, 64, 128, 24]), _log(rng, 1, 64)
        # no more bytes of rows, products or adapters than the largest listed case has
        while adapters > 1 and adapters * rank * (slices * k + n) > _MOST_WEIGHTS:
            adapters //= 2
        while batch * tokens > 1 and (batch * tokens * (k + 2 * n) > _MOST_ROWS
                                      or batch * tokens * rank * (slices * k + n) > _MOST_PRODUCTS):
            batch, tokens = (batch, tokens // 2) if tokens > 1 else (batch // 2, 1)
        return {"op": op, "batch": batch, "tokens": tokens, "k": k, "n": n, "rank": rank, "slices": slices, "adapters": adapters,
                "dtype": dtype}
    if op in ("rope", "rope_append"):
        heads, kv_heads, d = rng.choice(_HEADS if op == "rope_append" else _HEADS + _OTHER_HEADS)
        batch, tokens = _log(rng, 1, 64), rng.choice([1, _log(rng, 1, 4096)])
        tokens = max(1, min(tokens, _MOST_ROPE // (batch * (heads + 2 * kv_heads) * d)))
        axes = rng.choice([1, 1, 2, 3])
        return {"op": op, "batch": batch, "tokens": tokens, "ctx": rng.choice([rng.randint(0, 776), _log(rng, 1, 8192)]),
                "heads": heads, "kv_heads": kv_heads, "d": d, "rot": rng.choice([d, d, 16 * rng.randint(1, d // 16)]), "axes": axes,
                "mixed": axes > 1 and rng.random() < 0.5, "interleaved": rng.random() < 0.3, "norm": rng.random() < 0.7,
                "dtype": dtype}
    heads, kv_heads, d = rng.choice(_HEADS)
    batch = _log(rng, 1, 64)
    if op == "append":
        tokens = rng.choice([1, _log(rng, 1, 776)])
        tokens = max(1, min(tokens, 8 * 776 * 512 // (batch * 2 * kv_heads * d)))
        return {"op": op, "batch": batch, "tokens": tokens, "ctx": rng.randint(0, 776), "kv_heads": kv_heads, "d": d, "dtype": dtype}
    ctx = _log(rng, 1, 8192)
    tokens = min(ctx, rng.choice([1, 1, 1, _log(rng, 2, 64)]))
    # no more cached bytes than 64 x 8192 tokens of one head of 256
    batch = max(1, min(batch, 64 * 8192 * 256 // (ctx * kv_heads * d)))
    while tokens > 1 and batch * tokens * ctx * heads * d > 64 * 64 * 826 * 8 * 256:
        tokens //= 2
    return {"op": op, "batch": batch, "tokens": tokens, "ctx": ctx, "heads": heads, "kv_heads": kv_heads, "d": d,
            "causal": rng.random() < 0.7, "dtype": dtype}


# ------------------------------------------------------------------ inputs, from the seed
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(0x16B17 + int(seed))


def _activations(gen, *shape):
    x = torch.randn(shape, device="cuda", generator=gen)
    cols = torch.randperm(shape[-1], device="cuda", generator=gen)[: max(1, shape[-1] // 100)]
    x[..., cols] *= 20.0
    return x


def _cache(gen, case, pages_each):
    """A pool of pages in a random order: (k_cache, v_cache [P, KVH, 64, D], block_table [B, pages_each])."""
    b, kvh, d, t = case["batch"], case["kv_heads"], case["d"], DTYPES[case["dtype"]]
    n = b * pages_each
    table = torch.randperm(n, device="cuda", generator=gen).to(torch.int32).view(b, pages_each)
    sides = []
    for _ in range(2):
        side = torch.empty((n, kvh, PAGE, d), dtype=t, device="cuda")
        for p in range(0, n, 512):
            side[p:p + 512] = torch.randn((min(512, n - p), kvh, PAGE, d), device="cuda", generator=gen)
        sides.append(side)
    return *sides, table


def _lens(gen, batch, lo, hi):
    return torch.randint(lo, hi + 1, (batch,), device="cuda", generator=gen).to(torch.int32)


def _axis_of_pair(case):
    """The axis of each rotated pair: runs of pairs (a quarter for the first of three axes), or the axes in turn."""
    pairs, axes = case["rot"] // 2, case["axes"]
    if case["mixed"]:
        return [j % axes for j in range(pairs)]
    first = pairs // 4 if axes == 3 else pairs // axes
    rest = [first + (pairs - first) * i // max(axes - 1, 1) for i in range(axes)]
    return [sum(j >= edge for edge in rest[:axes - 1]) for j in range(pairs)]


def _positions(gen, case, start):
    """[axes, B, T]: one axis counts on from ``start``; several are text that counts on in all of them, with an image's grid in
    its middle half (time stands, height and width run)."""
    b, t, axes = case["batch"], case["tokens"], case["axes"]
    count = torch.arange(t, device="cuda")
    pos = (start[:, None] + count[None])[None].expand(axes, b, t).clone()
    if axes > 1 and t >= 16:
        lo, hi = t // 4, 3 * t // 4
        side = max(1, math.isqrt(hi - lo))
        grid = torch.arange(hi - lo, device="cuda")
        pos[:, :, lo:hi] = pos[:, :, lo:lo + 1]
        pos[-1, :, lo:hi] += grid % side
        pos[-2, :, lo:hi] += grid // side
    return (pos[0] if axes == 1 else pos).to(torch.int32).contiguous()


def _slice_widths(case):
    """Output columns of each part of a joined projection: heads of one KV head in three parts, else equal ones."""
    n, parts = case["n"], case["slices"]
    if parts == 3 and n == 2560:
        return [2048, 256, 256]
    return [n // parts] * parts


@torch.no_grad()
def prepare(case, seed):
    gen, op = _gen(seed), case["op"]
    t = DTYPES[case["dtype"]]
    b, tokens = case["batch"], case["tokens"]
    s = {"op": op, "t": t}
    if op == "lora":
        k, n, r, parts, count = case["k"], case["n"], case["rank"], case["slices"], case["adapters"]
        s["x"] = _activations(gen, b, tokens, k).to(t)
        s["y"] = _activations(gen, b, tokens, n).to(t)
        s["a"] = (torch.randn((count, parts * r, k), device="cuda", generator=gen) * k**-0.5).to(t)
        s["b"] = (torch.randn((count, n, r), device="cuda", generator=gen) * r**-0.5).to(t)
        s["scale"] = torch.rand((count,), device="cuda", generator=gen) + 0.5
        # every adapter has about as many requests; of eight requests or more, one in eight has none
        order = torch.randperm(b, device="cuda", generator=gen)
        ids = torch.arange(b, device="cuda") % count
        if b >= 8:
            ids[-(b // 8):] = -1
        s["ids"] = ids[order].to(torch.int32)
        s["widths"] = _slice_widths(case)
        return s
    kvh, d = case["kv_heads"], case["d"]
    if op == "attend":
        lo = max(tokens, case["ctx"] - (case["ctx"] // 2 if b > 1 else 0))
        s["lens"] = _lens(gen, b, lo, case["ctx"])
        s["kc"], s["vc"], s["table"] = _cache(gen, case, (case["ctx"] + PAGE - 1) // PAGE)
        s["q"] = (torch.randn((b, tokens, case["heads"], d), device="cuda", generator=gen) * 1.5).to(t)
        s["causal"], s["scaling"] = case["causal"], d**-0.5
        return s
    s["lens"] = _lens(gen, b, 3 * case["ctx"] // 4, case["ctx"])
    if op in ("rope_append", "append"):
        s["kc"], s["vc"], s["table"] = _cache(gen, case, case["ctx"] // PAGE + (tokens + 62) // PAGE + 2)
        s["counts"] = _lens(gen, b, max(1, tokens - tokens // 4), tokens)
    if op == "append":
        s["k"], s["v"] = (torch.randn((b, tokens, kvh, d), device="cuda", generator=gen).to(t) for _ in range(2))
        return s
    # views of the joined projection's output
    heads = case["heads"]
    joined = _activations(gen, b, tokens, (heads + 2 * kvh) * d).to(t).view(b, tokens, heads + 2 * kvh, d)
    s["q"], s["k"], s["v"] = joined[:, :, :heads], joined[:, :, heads:heads + kvh], joined[:, :, heads + kvh:]
    s["qw"], s["kw"] = ((torch.randn((d,), device="cuda", generator=gen) * 0.2).to(t) if case["norm"] else None for _ in range(2))
    half = case["rot"] // 2
    s["freq"] = (THETA ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)).float()
    s["pos"] = _positions(gen, case, s["lens"].long())
    s["axes"] = _axis_of_pair(case) if case["axes"] > 1 else None
    s["interleaved"] = case["interleaved"]
    return s


# ------------------------------------------------------------------ the calls
@torch.no_grad()
def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    from pi05_fast import w4a4

    op = s["op"]
    if op == "lora":
        return w4a4.lora_add(s["y"], s["x"], s["a"], s["b"], s["ids"], s["scale"], slices=s["widths"])
    if op == "rope":
        return w4a4.qk_norm_rope(s["q"], s["k"], s["qw"], s["kw"], EPS, s["pos"], s["freq"], interleaved=s["interleaved"],
                                 axes=s["axes"])
    if op == "rope_append":
        q = w4a4.qk_norm_rope_append(s["q"], s["k"], s["v"], s["qw"], s["kw"], EPS, s["pos"], s["freq"], s["kc"], s["vc"],
                                     s["table"], s["lens"], counts=s["counts"], interleaved=s["interleaved"], axes=s["axes"])
        return q, s["kc"], s["vc"]
    if op == "append":
        w4a4.kv_append(s["k"], s["v"], s["kc"], s["vc"], s["table"], s["lens"], counts=s["counts"])
        return s["kc"], s["vc"]
    return w4a4.kv_attention(s["q"], s["kc"], s["vc"], s["table"], s["lens"], s["scaling"], causal=s["causal"])


def _rope_plain(x, w, s):
    """Heads of x [B, T, H, D] behind their norm and rotation, in 32 bits."""
    f = x.float()
    if w is not None:
        f = f * (1.0 / torch.sqrt(f.square().mean(dim=-1, keepdim=True) + EPS)) * (1.0 + w.float())
    freq, pos = s["freq"].double(), s["pos"].double()
    if s["axes"] is not None:
        pos = pos[torch.tensor(s["axes"], device=x.device)].permute(1, 2, 0)  # [B, T, pairs]
    else:
        pos = pos[..., None]
    angle = (pos * freq)[:, :, None]
    c, sn = torch.cos(angle).float(), torch.sin(angle).float()
    half = freq.numel()
    if s["interleaved"]:
        a, b = f[..., 0:2 * half:2], f[..., 1:2 * half:2]
        turned = torch.stack((a * c - b * sn, b * c + a * sn), dim=-1).flatten(-2)
    else:
        a, b = f[..., :half], f[..., half:2 * half]
        turned = torch.cat((a * c - b * sn, b * c + a * sn), dim=-1)
    return torch.cat((turned, f[..., 2 * half:]), dim=-1).to(x.dtype)


def _append_plain(x, pool, s):
    """Writes the real tokens of x [B, T, KVH, D] behind the cached ones."""
    b, t = x.shape[:2]
    tok = torch.arange(t, device=x.device)[None].expand(b, t)
    real = tok < s["counts"][:, None]
    at = s["lens"].long()[:, None] + tok
    page = s["table"].long().gather(1, at // PAGE)
    pool[page[real], :, (at % PAGE)[real]] = x[real]


def _attend_plain(s):
    """q [B, T, H, D] over the gathered pages, in 32 bits."""
    q, lens, table = s["q"], s["lens"], s["table"].long()
    b, t, h, d = q.shape
    k, v = (c[table].float().transpose(1, 2).flatten(2, 3) for c in (s["kc"], s["vc"]))  # [B, KVH, L, D]
    kvh = k.size(1)
    rows = q.float().view(b, t, kvh, h // kvh, d).permute(0, 2, 1, 3, 4).reshape(b, kvh, t * (h // kvh), d)
    score = torch.matmul(rows, k.transpose(2, 3).contiguous()) * s["scaling"]
    tok = torch.arange(t, device=q.device).repeat_interleave(h // kvh)
    seen = lens[:, None] - t + tok[None] + 1 if s["causal"] else lens[:, None].expand(b, tok.numel())
    hidden = torch.arange(k.size(2), device=q.device)[None, None] >= seen[..., None]
    score = score.masked_fill_(hidden[:, None], float("-inf"))
    p = torch.exp(score - score.amax(dim=-1, keepdim=True))
    out = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    return out.view(b, kvh, t, h // kvh, d).permute(0, 2, 1, 3, 4).reshape(b, t, h, d).to(s["t"])


def _lora_plain(s):
    """All rows through all adapters; the rows' own products are kept and go through all second factors."""
    x, y, ids = s["x"], s["y"], s["ids"]
    count, n, r = s["b"].shape
    parts = len(s["widths"])
    m = x.numel() // x.size(-1)
    h = torch.matmul(x.reshape(m, -1).float(), s["a"].reshape(count * parts * r, -1).float().t()).view(m, count, parts, r)
    row = ids.long().repeat_interleave(m // ids.numel())
    mine = row[:, None] == torch.arange(count, device=x.device)[None]
    h = torch.where(mine[:, :, None, None], h * s["scale"][None, :, None, None], torch.zeros((), device=x.device))
    out, at = [], 0
    for g, width in enumerate(s["widths"]):
        w = s["b"][:, at:at + width].float().transpose(1, 2).reshape(count * r, width)
        out.append(y.reshape(m, n)[:, at:at + width].float() + torch.matmul(h[:, :, g].reshape(m, count * r), w))
        at += width
    return torch.cat(out, dim=1).view(y.shape).to(s["t"])


def _run_plain(s):
    op = s["op"]
    if op == "lora":
        return _lora_plain(s)
    if op == "attend":
        return _attend_plain(s)
    if op == "append":
        _append_plain(s["k"], s["kc"], s)
        _append_plain(s["v"], s["vc"], s)
        return s["kc"], s["vc"]
    q, k = _rope_plain(s["q"], s["qw"], s), _rope_plain(s["k"], s["kw"], s)
    if op == "rope":
        return q, k
    _append_plain(k, s["kc"], s)
    _append_plain(s["v"], s["vc"], s)
    return q, s["kc"], s["vc"]


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    op, b, t = case["op"], case["batch"], case["tokens"]
    if op == "lora":
        m, k, n, r, parts = b * t, case["k"], case["n"], case["rank"], case["slices"]
        used = min(case["adapters"], b - b // 8)
        real = m * (1 - (b // 8) / b)  # rows with an adapter: all of them are written, only these read x and are multiplied
        return {"bytes": 2.0 * (real * k + 2 * m * n + used * r * (parts * k + n)) + 4.0 * (b + used),
                "flops": 2.0 * real * r * (parts * k + n)}
    kvh, d = case["kv_heads"], case["d"]
    if op == "append":
        return {"bytes": 8.0 * b * t * kvh * d * 0.875, "flops": 0.0}
    if op in ("rope", "rope_append"):
        rows = b * t * (case["heads"] + kvh + (kvh * 0.875 if op == "rope_append" else 0))
        return {"bytes": 4.0 * rows * d + 4.0 * b * t * case["axes"], "flops": 10.0 * b * t * (case["heads"] + kvh) * d}
    length = case["ctx"] * (0.75 if b > 1 else 1.0)  # sequences of a batch are half to all of ctx
    return {"bytes": 4.0 * b * kvh * d * length + 4.0 * b * t * case["heads"] * d, "flops": 4.0 * b * case["heads"] * t * length * d}


# ------------------------------------------------------------------ 64-bit results
def _rope_exact(x, w, s):
    f64 = torch.float64
    y = x.to(f64)
    if w is not None:
        y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / y.size(-1) + EPS) * (w.to(f64) + 1)
    half = s["freq"].numel()
    first = torch.arange(half, device=x.device) * 2 if s["interleaved"] else torch.arange(half, device=x.device)
    second = first + 1 if s["interleaved"] else first + half
    out = y.clone()
    for j in range(half):
        pos = s["pos"] if s["axes"] is None else s["pos"][s["axes"][j]]
        turn = torch.polar(torch.ones((), dtype=f64, device=x.device), pos.to(f64) * s["freq"][j].to(f64))[..., None]
        z = torch.complex(y[..., first[j]], y[..., second[j]]) * turn
        out[..., first[j]], out[..., second[j]] = z.real, z.imag
    return out


@torch.no_grad()
def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    f64 = torch.float64
    if op == "lora":
        y = s["y"].to(f64)
        for i, which in enumerate(s["ids"].tolist()):
            if which < 0:
                continue
            at = 0
            for g, width in enumerate(s["widths"]):
                a = s["a"][which, g * case["rank"]:(g + 1) * case["rank"]].to(f64)
                h = s["x"][i].to(f64) @ a.t().contiguous() * s["scale"][which].to(f64)
                y[i, :, at:at + width] += h @ s["b"][which, at:at + width].to(f64).t().contiguous()
                at += width
        return y
    if op == "attend":
        out = torch.empty(s["q"].shape, dtype=f64, device="cuda")
        group = case["heads"] // case["kv_heads"]
        for i, length in enumerate(s["lens"].tolist()):
            ids = s["table"][i, : (length + PAGE - 1) // PAGE].long()
            for g in range(case["kv_heads"]):
                k, v = (c[ids, g].to(f64).reshape(-1, case["d"])[:length] for c in (s["kc"], s["vc"]))
                for h in range(g * group, (g + 1) * group):
                    z = (s["q"][i, :, h].to(f64).contiguous() @ k.t().contiguous()) * s["scaling"]
                    if s["causal"]:
                        last = length - case["tokens"] + torch.arange(case["tokens"], device="cuda")
                        z = z.masked_fill(torch.arange(length, device="cuda")[None] > last[:, None], float("-inf"))
                    out[i, :, h] = torch.softmax(z, dim=-1) @ v
        return out
    if op == "append":
        q, k, v = None, s["k"].to(f64), s["v"].to(f64)
    else:
        q, k, v = _rope_exact(s["q"], s["qw"], s), _rope_exact(s["k"], s["kw"], s), s["v"].to(f64)
        if op == "rope":
            return q, k
    pools = []
    for x, pool in ((k, s["kc"].to(f64)), (v, s["vc"].to(f64))):
        for i, (have, count) in enumerate(zip(s["lens"].tolist(), s["counts"].tolist())):
            at = 0
            while at < count:
                o = (have + at) % PAGE
                m = min(PAGE - o, count - at)
                pool[int(s["table"][i, (have + at) // PAGE]), :, o:o + m] = x[i, at:at + m].transpose(0, 1)
                at += m
        pools.append(pool)
    return tuple(pools) if q is None else (q, *pools)

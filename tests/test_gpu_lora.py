"""Low-rank adapters of many requests.

With small whole numbers every sum is exact in fp32 (below 2^24) and both 16-bit parts of h hold it, so that the
result is the exact sum rounded once: compared bit for bit.  With other numbers: h is within
K 2^-23 (|x| |a|^T) (K products, exact in fp32, summed in any order and with truncation at worst), its two
parts hold it to 2^-18 (bf16; fp16 2^-22, and 2^-38 of the row's largest), the second sum of R
products, twice over, is 2 R 2^-23 off, and the result half a step of its type and 2^-23 of its terms.
"""

from __future__ import annotations

import pytest
import torch

from pi05_fast import w4a4
from pi05_fast.w4a4 import extension as ext

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ids(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _ref(y, x, a, b, row_ids, scale, widths):
    """64-bit result and bound; rows [M, ...]."""
    r = b.size(2)
    out, tol = y.double().clone(), torch.zeros_like(y, dtype=torch.float64)
    part = 2.0**-18 if y.dtype == torch.bfloat16 else 2.0**-22
    for which in set(row_ids.tolist()):
        if not 0 <= which < a.size(0):
            continue
        rows = (row_ids == which).nonzero()[:, 0]
        s = 1.0 if scale is None else scale[which].double()
        at = 0
        for g, width in enumerate(widths):
            aa, bb = a[which, g * r:(g + 1) * r].double().t().contiguous(), b[which, at:at + width].double().t().contiguous()
            h, ha = x[rows].double() @ aa, x[rows].double().abs() @ aa.abs()
            out[rows, at:at + width] += s * (h @ bb)
            err = ha * (x.size(1) * 2.0**-23) + h.abs() * part + h.abs().amax(1, keepdim=True) * 2.0**-38
            tol[rows, at:at + width] += abs(s) * ((err + h.abs() * 2 * r * 2.0**-23) @ bb.abs()) * 1.01
            at += width
    tol += 2.0**-22 * (out.abs() + y.double().abs()) * (tol > 0)
    return out, tol + torch.finfo(y.dtype).eps / 2 * 1.001 * out.abs() * (tol > 0) + 2.0**-25 * (tol > 0)


def _whole(gen, m, k, n, r, adapters, parts, dtype):
    x = torch.zeros((m, k), device="cuda")
    x.scatter_(1, torch.randint(0, k, (m, 12), device="cuda", generator=gen), torch.randint(-2, 3, (m, 12), device="cuda", generator=gen).float())
    a = torch.randint(-2, 3, (adapters, parts * r, k), device="cuda", generator=gen)
    b = torch.randint(-2, 3, (adapters, n, r), device="cuda", generator=gen)
    y = torch.randint(-64, 65, (m, n), device="cuda", generator=gen)
    scale = torch.tensor([1.0, 0.5, -2.0, 0.0], device="cuda")[torch.arange(adapters, device="cuda") % 4]
    return [t.to(dtype) for t in (y, x, a, b)] + [scale]


def _exact(y, x, a, b, row_ids, scale, widths):
    return _ref(y, x, a, b, row_ids, scale, widths)[0].to(torch.float32).to(y.dtype)


SHAPES = [(1, 64, 8, 8, 1, 1), (1, 2048, 2560, 16, 5, 3), (3, 104, 33, 24, 2, 1), (17, 2048, 130, 8, 30, 2), (64, 512, 2048, 16, 64, 1),
          (40, 1000, 999, 40, 7, 1), (200, 264, 192, 64, 3, 3), (33, 16384, 64, 128, 4, 4), (700, 128, 257, 32, 6, 1), (257, 40, 96, 128, 2, 2),
          (40, 4104, 320, 64, 5, 1), (20, 16384, 130, 24, 3, 1), (1, 16384, 96, 16, 2, 3), (300, 2048, 1100, 16, 40, 1)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n,r,adapters,parts", SHAPES)
def test_whole_numbers(cuda, m, k, n, r, adapters, parts, dtype):
    """Rows in any order, in runs, all of one adapter, and without one; new outputs and in place."""
    gen = _gen(m + k + n + r)
    y, x, a, b, scale = _whole(gen, m, k, n, r, adapters, parts, dtype)
    widths = [n // parts] * parts if parts != 3 or n != 2560 else [2048, 256, 256]
    slices = None if parts == 1 else widths
    for ids in (torch.randint(-1, adapters + 1, (m,), device="cuda", generator=gen), torch.arange(m, device="cuda") * adapters // m,
                torch.full((m,), adapters - 1, device="cuda"), torch.full((m,), -1, device="cuda")):
        ids = ids.to(torch.int32)
        want = _exact(y, x, a, b, ids, scale, widths)
        got = w4a4.lora_add(y, x, a, b, ids, scale, slices=slices)
        assert torch.equal(got, want)
        z = y.clone()
        assert w4a4.lora_add_(z, x, a, b, ids, scale, slices=slices) is z and torch.equal(z, want)
        one = _exact(y, x, a, b, ids, None, widths)
        assert torch.equal(w4a4.lora_add(y, x, a, b, ids, slices=slices), one)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n,r,adapters", [(1, 64, 64, 16, 1), (50, 2048, 300, 16, 12), (130, 256, 2048, 64, 3), (16, 16384, 2048, 8, 16)])
def test_values(cuda, m, k, n, r, adapters, dtype):
    gen = _gen(m + k)
    y, x = (torch.randn((m, w), device="cuda", generator=gen).to(dtype) for w in (n, k))
    x[:, ::97] *= 20
    a = (torch.randn((adapters, r, k), device="cuda", generator=gen) * k**-0.5).to(dtype)
    b = (torch.randn((adapters, n, r), device="cuda", generator=gen) * r**-0.5).to(dtype)
    scale = torch.rand(adapters, device="cuda", generator=gen) + 0.5
    ids = torch.randint(-1, adapters, (m,), device="cuda", generator=gen).to(torch.int32)
    got = w4a4.lora_add(y, x, a, b, ids, scale)
    want, tol = _ref(y, x, a, b, ids, scale, [n])
    assert ((got.double() - want).abs() <= tol).all(), ((got.double() - want).abs() / tol.clamp_min(1e-30)).max().item()


def test_requests_of_many_tokens(cuda):
    """An id for each request of a padded batch, for each token, and one for all."""
    gen = _gen(1)
    y, x, a, b, scale = _whole(gen, 4 * 50, 256, 96, 16, 3, 1, torch.float16)
    y, x = y.view(4, 50, 96), x.view(4, 50, 256)
    ids = _ids([2, -1, 0, 1])
    flat = ids.repeat_interleave(50)
    want = _exact(y.view(200, 96), x.view(200, 256), a, b, flat, scale, [96]).view(4, 50, 96)
    assert torch.equal(w4a4.lora_add(y, x, a, b, ids, scale), want)
    assert torch.equal(w4a4.lora_add(y, x, a, b, flat.view(4, 50), scale), want)
    one = _exact(y.view(200, 96), x.view(200, 256), a, b, torch.full_like(flat, 2), scale, [96]).view(4, 50, 96)
    assert torch.equal(w4a4.lora_add(y, x, a, b, _ids(2), scale), one)


@pytest.mark.parametrize("adapters", [1, 3, 70])
@pytest.mark.parametrize("per_id", [1, 2, 5, 16, 31, 63, 64, 65, 100, 130])
def test_requests_of_any_length(cuda, per_id, adapters):
    """Rows of an adapter together or apart, fewer and more than a tile, and rows of NaN beside them."""
    requests = 200 // per_id + 2
    m = requests * per_id
    gen = _gen(per_id + adapters)
    y, x, a, b, scale = _whole(gen, m, 72, 40, 8, adapters, 1, torch.bfloat16)
    bad = torch.zeros(m, dtype=torch.bool, device="cuda")
    bad[::7] = True
    for ids in (torch.randint(-1, adapters + 1, (requests,), device="cuda", generator=gen), torch.arange(requests, device="cuda") % 3 - 1):
        ids = ids.to(torch.int32)
        rows = ids.repeat_interleave(per_id)
        want = _exact(y, x, a, b, rows, scale, [40])
        xs = x.masked_fill(bad[:, None], float("nan")).view(requests, per_id, 72)
        got = w4a4.lora_add(y.view(requests, per_id, 40), xs, a, b, ids, scale).view(m, 40)
        named = (rows >= 0) & (rows < adapters)
        assert torch.equal(got[~bad | ~named], want[~bad | ~named]) and torch.isnan(got[bad & named]).all()
        z = y.clone().view(requests, per_id, 40)
        w4a4.lora_add_(z, xs, a, b, ids, scale)
        assert torch.equal(z.view(m, 40).nan_to_num(0), got.nan_to_num(0))


def test_rows_short_of_a_request(cuda):
    """At the C entry the last id may have fewer rows than the others."""
    lib = ext.load_int4_gemm()
    for m, per_id in ((150, 64), (37, 20), (129, 128), (5, 9)):
        y, x, a, b, scale = _whole(_gen(m), m, 64, 48, 16, 3, 1, torch.float16)
        ids = torch.arange((m + per_id - 1) // per_id, device="cuda").to(torch.int32) % 3
        out, ws = torch.empty_like(y), torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
        assert lib.pi05w4a4_lora_workspace_bytes(m, per_id, 64, 48, 16, 1, 3) <= ws.numel()
        rc = lib.pi05w4a4_lora_add(y.data_ptr(), 48, x.data_ptr(), 64, m, 64, a.data_ptr(), b.data_ptr(), scale.data_ptr(), 3, 16, ids.data_ptr(),
                                   per_id, 48, 1, None, 0, out.data_ptr(), 48, ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream)
        assert rc == 0 and torch.equal(out, _exact(y, x, a, b, ids.repeat_interleave(per_id)[:m], scale, [48]))


def test_many_rows_of_a_long_k(cuda):
    """K in slices although every CU has rows."""
    y, x, a, b, scale = _whole(_gen(10), 5000, 16384, 64, 24, 2, 1, torch.float16)
    ids = torch.arange(50, device="cuda").to(torch.int32) % 3
    want = _exact(y, x, a, b, ids.repeat_interleave(100), scale, [64])
    assert torch.equal(w4a4.lora_add(y.view(50, 100, 64), x.view(50, 100, 16384), a, b, ids, scale).view(5000, 64), want)


def test_strides(cuda):
    """Parts of wider rows, at any element, written in place; nothing beside them changes."""
    gen = _gen(2)
    y, x, a, b, scale = _whole(gen, 37, 128, 100, 8, 4, 1, torch.bfloat16)
    ids = torch.randint(-1, 4, (37,), device="cuda", generator=gen).to(torch.int32)
    want = _exact(y, x, a, b, ids, scale, [100])
    for at, width in ((0, 104), (3, 211), (8, 128), (16, 301)):
        wide = torch.full((37, width), 7.0, device="cuda", dtype=torch.bfloat16)
        wide[:, at:at + 100] = y
        assert torch.equal(w4a4.lora_add(wide[:, at:at + 100], x, a, b, ids, scale), want)
        w4a4.lora_add_(wide[:, at:at + 100], x, a, b, ids, scale)
        assert torch.equal(wide[:, at:at + 100], want) and (wide[:, :at] == 7).all() and (wide[:, at + 100:] == 7).all()
    xw = torch.randn((37, 300), device="cuda", generator=gen).bfloat16()
    for at in (0, 8, 5):
        xw[:, at:at + 128] = x
        assert torch.equal(w4a4.lora_add(y, xw[:, at:at + 128], a, b, ids, scale), want)
    assert torch.equal(w4a4.lora_add(y.t().contiguous().t(), x, a, b, ids, scale), want)
    assert torch.equal(w4a4.lora_add(y, x, a, b.transpose(1, 2).contiguous().transpose(1, 2), ids, scale), want)
    rows = y[:1].expand(37, 100)
    assert torch.equal(w4a4.lora_add(rows, x, a, b, ids, scale), _exact(rows.contiguous(), x, a, b, ids, scale, [100]))
    # the projection's input is its output too, or lies in the same rows
    b2 = torch.randint(-2, 3, (4, 128, 8), device="cuda", generator=gen).bfloat16()
    for _ in range(5):
        sq = x.clone()
        w4a4.lora_add_(sq, sq, a, b2, ids, scale)
        assert torch.equal(sq, _exact(x, x, a, b2, ids, scale, [128]))
    both = torch.cat((y, torch.zeros_like(y)[:, :4], x), dim=1)
    w4a4.lora_add_(both[:, :100], both[:, 104:], a, b, ids, scale)
    assert torch.equal(both[:, :100], want) and torch.equal(both[:, 104:], x)


def test_what_is_not_finite_stays_in_its_rows(cuda):
    gen = _gen(3)
    for dtype in TYPES:
        y, x, a, b, scale = _whole(gen, 40, 128, 160, 16, 5, 1, dtype)
        ids = torch.arange(40, device="cuda", dtype=torch.int32) % 6 - 1
        want = _exact(y, x, a, b, ids, None, [160])
        x[7, 3], x[20, 5] = float("nan"), float("inf")
        a[4], b[3, :, 2] = float("nan"), float("inf")
        got = w4a4.lora_add(y, x, a, b, ids)
        touched = (ids == 4) | (ids == 3)
        touched[7] = touched[20] = True
        assert torch.equal(got[~touched], want[~touched]) and not torch.isfinite(got[ids == 4]).any()
        assert torch.isnan(got[7]).any() and not torch.isfinite(got[ids == 3]).all()


def test_range_of_h(cuda):
    """Sums between the two products that fp16 does not hold, either way."""
    gen = _gen(4)
    for scale_a, scale_b in ((200.0, 2.0**-14), (2.0**-13, 100.0)):
        x = torch.randn((20, 512), device="cuda", generator=gen).half() * 100
        a = (torch.randn((2, 16, 512), device="cuda", generator=gen) * scale_a).half()
        b = (torch.randn((2, 64, 16), device="cuda", generator=gen) * scale_b).half()
        if scale_a < 1:
            x = (x * 1e-4).half()
        y = torch.randn((20, 64), device="cuda", generator=gen).half()
        ids = torch.arange(20, device="cuda", dtype=torch.int32) % 2
        got = w4a4.lora_add(y, x, a, b, ids)
        want, tol = _ref(y, x, a, b, ids, None, [64])
        assert torch.isfinite(got).all() and ((got.double() - want).abs() <= tol).all()


def test_weights_past_4_gib(cuda):
    gen = _gen(5)
    count = 70000
    a = torch.zeros((count, 16, 2048), dtype=torch.float16, device="cuda")  # 4.6 GB
    b = torch.zeros((count, 2080, 16), dtype=torch.float16, device="cuda")
    y, x, a1, b1, _ = _whole(gen, 20, 2048, 2080, 16, 2, 1, torch.float16)
    a[-1], a[69000], b[-1], b[69000] = a1[0], a1[1], b1[0], b1[1]
    ids = torch.arange(20, device="cuda", dtype=torch.int32) % 2
    far = torch.where(ids == 0, count - 1, 69000).to(torch.int32)
    assert torch.equal(w4a4.lora_add(y, x, a, b, far), w4a4.lora_add(y, x, a1, b1, ids))


def test_streams_and_graphs(cuda):
    gen = _gen(6)
    sets = [_whole(gen, 32, 2048, 512, 16, 8, 1, torch.float16) for _ in range(2)]
    ids = torch.randint(-1, 8, (32,), device="cuda", generator=gen).to(torch.int32)
    wants = [_exact(s[0], s[1], s[2], s[3], ids, s[4], [512]) for s in sets]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i in range(10):
        with torch.cuda.stream(streams[i % 2]):
            s = sets[i % 2]
            got.append(w4a4.lora_add(s[0], s[1], s[2], s[3], ids, s[4]))
    torch.cuda.synchronize()
    assert all(torch.equal(g, wants[i % 2]) for i, g in enumerate(got))
    graphs = []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = w4a4.lora_add(s[0], s[1], s[2], s[3], ids, s[4])
        graphs.append((g, out))
    for i in range(6):
        new = torch.randint(-1, 8, (32,), device="cuda", generator=gen).to(torch.int32)
        ids.copy_(new)
        for (g, out), s in zip(graphs, sets):
            out.zero_()
            g.replay()
            eager = w4a4.lora_add(s[0], s[1], s[2], s[3], ids, s[4])
            torch.cuda.synchronize()
            assert torch.equal(out, eager) and torch.equal(out, _exact(s[0], s[1], s[2], s[3], ids, s[4], [512]))


def test_refusals(cuda):
    y, x, a, b, scale = _whole(_gen(7), 4, 64, 32, 8, 2, 1, torch.float16)
    ids = _ids([0, 1, -1, 0])

    def call(y=y, x=x, a=a, b=b, ids=ids, scale=scale, fn=w4a4.lora_add, **kw):
        return fn(y, x, a, b, ids, scale, **kw)

    for kw, text in [
        (dict(y=y.float()), "of one type"), (dict(x=x.bfloat16()), "of one type"), (dict(a=a.float()), "of one type"), (dict(x=x[:3]), "same rows"),
        (dict(x=x[None]), "same rows"), (dict(a=a[:1]), "expects a"), (dict(b=b[:, :16]), "expects a"), (dict(a=a[:, :4]), "expects a"),
        (dict(a=a[..., :32]), "expects a"), (dict(slices=[16, 16]), "expects a"), (dict(slices=[16, 8]), "slices"), (dict(slices=[32, 0]), "slices"),
        (dict(slices=[]), "slices"), (dict(slices=[8, 8, 8, 4, 4]), "slices"), (dict(ids=ids.long()), "ids"), (dict(ids=ids[:3]), "ids"),
        (dict(ids=ids[:, None]), "ids"), (dict(ids=ids.cpu()), "must be on"), (dict(scale=scale.half()), "scale"), (dict(scale=scale[:1]), "scale"),
        (dict(x=x[:, :60], a=a[..., :60].contiguous()), "multiples of 8"), (dict(a=a[:, :4].contiguous(), b=b[..., :4].contiguous()), "multiples of 8"),
        (dict(y=y[:1].expand(4, 32), fn=w4a4.lora_add_), "rows of y"), (dict(y=y.t().contiguous().t(), fn=w4a4.lora_add_), "rows of y"),
    ]:
        with pytest.raises(RuntimeError, match=text):
            call(**kw)
    assert call(y=y[:0], x=x[:0], ids=ids[:0]).shape == (0, 32)
    assert torch.equal(call(a=a[:0], b=b[:0], scale=scale[:0]), y)
    assert call(y=y[:, :0], b=b[:, :0]).shape == (4, 0)
    leaf = x.clone().requires_grad_()
    with pytest.raises((RuntimeError, NotImplementedError)):
        call(x=leaf).sum().backward()


@pytest.mark.filterwarnings("ignore:There is a performance drop")
def test_vmap(cuda):
    y, x, a, b, scale = _whole(_gen(9), 6, 64, 48, 8, 2, 1, torch.float16)
    y, x, ids = y.view(3, 2, 48), x.view(3, 2, 64), _ids([0, 1, -1])
    assert torch.equal(torch.vmap(lambda y, x, i: w4a4.lora_add(y, x, a, b, i, scale))(y, x, ids), w4a4.lora_add(y, x, a, b, ids, scale))
    with pytest.raises(RuntimeError):
        torch.vmap(lambda y, x, i: w4a4.lora_add_(y, x, a, b, i, scale))(y, x, ids)


def test_dispatched_route(cuda):
    y, x, a, b, scale = _whole(_gen(8), 5, 64, 48, 8, 2, 2, torch.float16)
    ids = _ids([0, 1, -1, 0, 1])

    def step(y, x):
        z = w4a4.lora_add(y, x, a, b, ids, scale, slices=[16, 32])
        w4a4.lora_add_(z[:, 16:], x, a[:, :8], b[:, 16:], ids, scale)
        return z

    want = step(y, x)
    assert torch.equal(torch.compile(step, fullgraph=True, backend="eager")(y, x), want)

"""int8 rows and int8 products against their definitions in 64 bits.

Tolerances.  h = 2^-24 is an fp32 half step, u(T) = finfo(T).eps / 2 one of the output type.
* Behind a norm: the sum of K squares is made of per-thread runs of at most 32, 6 steps across a
  wave and 15 across waves, so it is within 53 h, its square root within 27 h; division by K,
  eps, root, reciprocal, weight, products and the scale's own division add less than 20 h.  A code's
  argument is then within 127 * 64 h = 5e-4 of the true one.
* A product: the sums are exact, their conversion, two scalings and two additions are one h
  each of what they add up, then u(T) of the result (2^-25 absolutely below fp16's normal range).
"""

from __future__ import annotations

import pytest
import torch

from pi05_fast.w4a4 import int8 as i8

pytestmark = pytest.mark.gpu
H = 2.0**-24
TYPES = [torch.float16, torch.bfloat16]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _x(gen, m, k, t):
    x = torch.randn((m, k), device="cuda", generator=gen)
    x[:, torch.randperm(k, device="cuda", generator=gen)[: max(1, k // 100)]] *= 20
    return x.to(t)


def _check_rows(y, q, s):
    """q, s against rows y (float64)."""
    amax = y.abs().amax(-1)
    assert ((s.double() - (amax / 127 + 1e-12)).abs() <= 64 * H * (amax / 127) + H * 1e-12).all()
    off = (q.double() - y / s.double()[:, None]).abs()
    assert off.max().item() <= 0.5 + 127 * 64 * H
    assert q.abs().max().item() <= 127


ROWS = [(1, 8), (1, 2048), (3, 64), (5, 1000), (7, 2056), (64, 2048), (517, 2048), (1100, 512), (600, 1992), (9, 8192), (4, 8200),
        (3, 16384), (2, 32768), (700, 1024)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,k", ROWS)
def test_quantize_is_exact(cuda, m, k, t):
    """Codes and scales of plain rows are those of the fp32 definition, bit for bit."""
    x = _x(_gen(m * 31 + k), m, k, t)
    q, s = i8.quantize_int8(x)
    c = x.cpu().float()
    scale = c.abs().amax(-1) / torch.full((m,), 127.0) + 1e-12
    want = torch.round(c.double() * (1.0 / scale).double()[:, None])
    assert torch.equal(s.cpu(), scale)
    assert torch.equal(q.cpu().double(), want)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,k", ROWS)
@pytest.mark.parametrize("unit", [True, False])
def test_norm_forms(cuda, m, k, t, unit):
    gen = _gen(m * 17 + k)
    x, r = _x(gen, m, k, t), _x(gen, m, k, t)
    w = (torch.randn((k,), device="cuda", generator=gen) * 0.2 + (0 if unit else 1)).to(t)
    g = w.double() + (1 if unit else 0)
    for h, got in ((x, i8.rms_norm_int8(x, w, 1e-6, unit)), (x + r, i8.add_rms_norm_int8(x, r, w, 1e-6, unit))):
        hd = h.double()
        _check_rows(hd / (hd.square().mean(-1, keepdim=True) + 1e-6).sqrt() * g, got[0], got[1])
        if len(got) == 3:
            assert torch.equal(got[2], h)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,k", [(4, 2048), (1100, 2048), (4, 32768)])
def test_rows_zeros_and_nonfinite(cuda, m, k, t):
    x = torch.randn((m, k), device="cuda", generator=_gen(1)).to(t)
    x[0] = 0
    x[1, k - 1] = float("nan")
    x[2, 0] = float("-inf")
    w = torch.zeros(k, device="cuda", dtype=t)
    for q, s in (i8.quantize_int8(x), i8.rms_norm_int8(x, w, 1e-6), i8.add_rms_norm_int8(x, torch.zeros_like(x), w, 1e-6)[:2]):
        assert s[0].item() == pytest.approx(1e-12) and not q[0].any()
        assert torch.isnan(s[1:3]).all() and not q[1:3].any()
        assert torch.isfinite(s[3:]).all() and q[3:].any()


def test_rows_strides_alignment_and_empty(cuda):
    gen = _gen(5)
    wide = _x(gen, 33, 2560, torch.float16)
    for x in (wide[:, 512:768], wide[:, 4:260], wide[::2, :256], wide.t()[:2560, :32]):
        q, s = i8.quantize_int8(x)
        q2, s2 = i8.quantize_int8(x.contiguous())
        assert torch.equal(q, q2) and torch.equal(s, s2)
    w = _x(gen, 1, 264, torch.float16)[0]
    a = i8.add_rms_norm_int8(wide[:, :256], wide[:, 1024:1280], w[8:], 1e-6)
    b = i8.add_rms_norm_int8(wide[:, :256].contiguous(), wide[:, 1024:1280].contiguous(), w[8:].clone(), 1e-6)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    q, s = i8.quantize_int8(wide[:0])
    assert q.shape == (0, 2560) and s.shape == (0,)
    q, s = i8.quantize_int8(wide.view(3, 11, 2560))
    assert q.shape == (3, 11, 2560) and s.shape == (3, 11)


def test_rows_far_offsets(cuda):
    """Rows behind 2^31 elements."""
    m, k = 70000, 32768
    x = torch.empty((m, k), dtype=torch.bfloat16, device="cuda")
    x[:8] = 1
    tail = _x(_gen(2), 8, k, torch.bfloat16)
    x[-8:] = tail
    q, s = i8.quantize_int8(x)
    q2, s2 = i8.quantize_int8(tail)
    assert torch.equal(q[-8:], q2) and torch.equal(s[-8:], s2) and (q[:8] == 127).all()


# ------------------------------------------------------------------ product
def _product(gen, m, k, n, t, bias, res):
    q = torch.randint(-127, 128, (m, k), device="cuda", generator=gen, dtype=torch.int8)
    w = torch.randint(-128, 128, (n, k), device="cuda", generator=gen, dtype=torch.int8)
    sq = torch.rand((m,), device="cuda", generator=gen) * 0.02 + 1e-3
    sw = torch.rand((n,), device="cuda", generator=gen) * 2e-3 + 1e-4
    return (q, sq, w, sw, torch.randn((n,), device="cuda", generator=gen).to(t) if bias else None,
            torch.randn((m, n), device="cuda", generator=gen).to(t) if res else None)


def _check_product(y, q, sq, w, sw, bias, res):
    t = y.dtype
    p = (q.double() @ w.double().t().contiguous()) * sq.double()[:, None] * sw.double()
    want, mag = p.clone(), p.abs()
    for e in (bias, res):
        if e is not None:
            want += e.double()
            mag += e.double().abs()
    tol = 6 * H * mag + (torch.finfo(t).eps / 2) * (1 + 1e-3) * want.abs() + 2.0**-25
    over = want.abs() > torch.finfo(t).max
    assert (((y.double() - want).abs() <= tol) | over).all()


PRODUCTS = [(1, 16, 1), (1, 2048, 2560), (2, 64, 7), (5, 16384, 33), (15, 80, 100), (16, 144, 64), (17, 2048, 40), (33, 272, 65),
            (48, 4096, 130), (64, 2048, 2048), (65, 2048, 257), (100, 16, 17), (127, 128, 128), (129, 208, 129), (256, 2064, 300),
            (300, 144, 5), (513, 1024, 1000), (776, 2048, 2560), (1000, 4096, 1016), (1030, 16384, 136), (2111, 512, 2047),
            (3, 65536, 24), (300, 65536, 40)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,k,n", PRODUCTS)
def test_product(cuda, m, k, n, t):
    gen = _gen(m + 7 * k + n)
    for bias, res in ((False, False), (True, True)):
        args = _product(gen, m, k, n, t, bias, res)
        _check_product(i8.int8_gemm(*args[:4], bias=args[4], residual=args[5], out_dtype=t), *args)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,k,n", [(4200, 1040, 4200), (8192, 112, 8201), (2600, 16, 2568), (4100, 2048, 4097),
                                   (4100, 272, 4160), (3355, 256, 2624)])
def test_product_of_many_tiles(cuda, m, k, n, t):
    """More large tiles than CUs, the last of a row, column and K ragged, and K of a single step."""
    q, sq, w, sw, bias, res = _product(_gen(m + k + n), m, k, n, t, True, True)
    y = i8.int8_gemm(q, sq, w, sw, bias, res, out_dtype=t)
    plain = i8.int8_gemm(q, sq, w, sw, out_dtype=t)
    for r in range(0, m, 1024):  # rows at a time: the 64-bit products
        part = slice(r, r + 1024)
        _check_product(y[part], q[part], sq[part], w, sw, bias, res[part])
        _check_product(plain[part], q[part], sq[part], w, sw, None, None)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,k,n", [(4, 16384, 67), (70, 16384, 67), (200, 8192, 129), (900, 512, 771), (300, 256, 2), (5000, 256, 4099)])
def test_product_of_odd_rows(cuda, m, k, n, t):
    """Output rows, K slices and residual rows that begin at any element."""
    q, sq, w, sw, bias, res = _product(_gen(m + n), m, k, n, t, True, True)
    want = i8.int8_gemm(q, sq, w, sw, bias, res, out_dtype=t)
    _check_product(want, q, sq, w, sw, bias, res)
    wide = torch.zeros((m, n + 6), dtype=t, device="cuda")
    wide[:, 3:n + 3] = res
    odd_bias = torch.zeros(n + 1, dtype=t, device="cuda")
    odd_bias[1:] = bias
    assert torch.equal(i8.int8_gemm(q, sq, w, sw, odd_bias[1:], wide[:, 3:n + 3], out_dtype=t), want)


def test_product_of_more_rows_than_a_launch_has_tiles(cuda):
    m, k, n = (1 << 30) + 100, 16, 8
    q = torch.empty((m, k), dtype=torch.int8, device="cuda")
    sq = torch.empty((m,), device="cuda")
    at = [slice(0, 300), slice(m // 2 - 150, m // 2 + 150), slice(m - 300, m)]
    gen = _gen(5)
    parts = [_product(gen, 300, k, n, torch.float16, False, False) for _ in at]
    for s, p in zip(at, parts):
        q[s], sq[s] = p[0], p[1]
    y = i8.int8_gemm(q, sq, *parts[0][2:4])
    for s, p in zip(at, parts):
        _check_product(y[s], p[0], p[1], *parts[0][2:4], None, None)


@pytest.mark.parametrize("m,n", [(1, 64), (40, 200), (300, 300), (700, 1024)])
def test_product_extreme_sums(cuda, m, n):
    """The largest sum that K = 65536 can make, 2^30, is exact."""
    k = 65536
    q = torch.full((m, k), -128, dtype=torch.int8, device="cuda")
    w = torch.full((n, k), -128, dtype=torch.int8, device="cuda")
    sq, sw = torch.full((m,), 2.0**-20, device="cuda"), torch.full((n,), 2.0**-3, device="cuda")
    assert (i8.int8_gemm(q, sq, w, sw) == 128).all()


@pytest.mark.parametrize("m", [3, 50, 200, 900])
def test_product_strides_and_alignment(cuda, m):
    gen = _gen(m)
    q, sq, w, sw, bias, res = _product(gen, m, 1024, 136, torch.float16, True, True)
    want = i8.int8_gemm(q, sq, w, sw, bias, res)
    wide_q, wide_w = torch.zeros((m, 1536), dtype=torch.int8, device="cuda"), torch.zeros((136, 1280), dtype=torch.int8, device="cuda")
    wide_q[:, 256:1280], wide_w[:, 16:1040] = q, w
    odd_q = torch.zeros((m, 1029), dtype=torch.int8, device="cuda")
    odd_q[:, 3:1027] = q
    wide_r = torch.zeros((m, 301), dtype=torch.float16, device="cuda")
    wide_r[:, 5:141] = res
    assert torch.equal(i8.int8_gemm(wide_q[:, 256:1280], sq, wide_w[:, 16:1040], sw, bias, res), want)
    assert torch.equal(i8.int8_gemm(odd_q[:, 3:1027], sq, w, sw, bias, wide_r[:, 5:141]), want)
    assert torch.equal(i8.int8_gemm(q.view(1, m, 1024), sq.view(1, m), w, sw, bias, res.view(1, m, 136)), want.view(1, m, 136))


def test_product_nan_scales_stay_in_their_rows(cuda):
    for m in (4, 300):
        q, sq, w, sw, _, _ = _product(_gen(m), m, 256, 96, torch.float16, False, False)
        want = i8.int8_gemm(q, sq, w, sw)
        sq2 = sq.clone()
        sq2[1] = float("nan")
        got = i8.int8_gemm(q, sq2, w, sw)
        assert torch.isnan(got[1]).all() and torch.equal(got[[0, 2, 3]], want[[0, 2, 3]])


def test_product_does_not_write_outside(cuda):
    """The rows around an output that a caller carves out of a larger buffer keep their values."""
    lib = i8.load_int4_gemm()
    for m, n in ((5, 24), (70, 40), (300, 72), (1000, 1032)):
        k = 256
        q, sq, w, sw, _, _ = _product(_gen(m), m, k, n, torch.float16, False, False)
        buf = torch.full(((m + 64) * n,), 7.0, dtype=torch.float16, device="cuda")
        y = buf[32 * n:(32 + m) * n]
        need = lib.pi05w4a4_int8_gemm_workspace_bytes(m, n, k)
        ws = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
        assert lib.pi05w4a4_int8_gemm(q.data_ptr(), k, sq.data_ptr(), m, k, w.data_ptr(), k, sw.data_ptr(), n, None, None, 0, 0,
                                      y.data_ptr(), ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream) == 0
        assert torch.equal(y.view(m, n), i8.int8_gemm(q, sq, w, sw))
        assert (buf[: 32 * n] == 7).all() and (buf[(32 + m) * n:] == 7).all()


def test_product_far_offsets(cuda):
    """Operands and outputs behind 2^32 bytes."""
    m, k, n = 140000, 16384, 16
    q = torch.zeros((m, 32768), dtype=torch.int8, device="cuda")
    q[-3:, :k] = torch.randint(-127, 128, (3, k), device="cuda", generator=_gen(1), dtype=torch.int8)
    w = torch.randint(-127, 128, (n, k), device="cuda", generator=_gen(2), dtype=torch.int8)
    sq, sw = torch.full((m,), 1e-3, device="cuda"), torch.full((n,), 1e-3, device="cuda")
    got = i8.int8_gemm(q[:, :k], sq, w, sw)
    assert not got[:-3].any()
    _check_product(got[-3:], q[-3:, :k], sq[-3:], w, sw, None, None)


def test_refusals_on_the_gpu(cuda):
    x = torch.zeros((4, 64), dtype=torch.float16, device="cuda")
    q, s = i8.quantize_int8(x)
    w, sw = i8.quantize_int8(torch.zeros((8, 64), dtype=torch.float16, device="cuda"))
    bad = [
        (lambda: i8.quantize_int8(x.float()), "float16 or bfloat16"),
        (lambda: i8.quantize_int8(x[:, :12]), "multiple of 8"),
        (lambda: i8.rms_norm_int8(x, x[0, :32], 1e-6), "norm weight"),
        (lambda: i8.rms_norm_int8(x, x[0].bfloat16(), 1e-6), "norm weight"),
        (lambda: i8.rms_norm_int8(x, x[0].cpu(), 1e-6), "norm weight"),
        (lambda: i8.add_rms_norm_int8(x, x[:2], x[0], 1e-6), "residual"),
        (lambda: i8.int8_gemm(q, s, w, sw, out_dtype=torch.float32), "writes float16"),
        (lambda: i8.int8_gemm(x, s, w, sw), "int8 codes"),
        (lambda: i8.int8_gemm(q, s[:3], w, sw), "q_scale"),
        (lambda: i8.int8_gemm(q, s, w, sw.half()), "w_scale"),
        (lambda: i8.int8_gemm(q, s.cpu(), w, sw), "q_scale"),
        (lambda: i8.int8_gemm(q, s, w[:, :48], sw), "K=64"),
        (lambda: i8.int8_gemm(q[:, :24], s, w[:, :24], sw), "multiple of 16"),
        (lambda: i8.int8_gemm(q, s, w.cpu(), sw), "weights must be on"),
        (lambda: i8.int8_gemm(q, s, w, sw, bias=x[0, :7]), "bias"),
        (lambda: i8.int8_gemm(q, s, w, sw, residual=x), "residual"),
        (lambda: i8.int8_gemm(q, s, w, sw, residual=x[:, :8].bfloat16()), "residual"),
    ]
    for call, text in bad:
        with pytest.raises(RuntimeError, match=text):
            call()


def test_graph_replays(cuda):
    """A captured norm + product pair follows its inputs over replays, split K and tiles among them."""
    for m, k, n in ((3, 16384, 64), (200, 1024, 300)):
        gen = _gen(m)
        x, w = _x(gen, m, k, torch.float16), torch.zeros(k, dtype=torch.float16, device="cuda")
        wq, sw = i8.quantize_int8(_x(gen, n, k, torch.float16))

        def run(src):
            q, s, h = i8.add_rms_norm_int8(src, src, w, 1e-6)
            return i8.int8_gemm(q, s, wq, sw), h

        static = x.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run(static)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run(static)
        for i in range(4):
            src = _x(gen, m, k, torch.float16)
            static.copy_(src)
            graph.replay()
            want = run(src)
            torch.cuda.synchronize()
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_two_streams_at_once(cuda):
    """Split-K calls on two streams have workspaces of their own."""
    gen = _gen(9)
    args = [_product(gen, 8, 16384, 128, torch.float16, False, False)[:4] for _ in range(2)]
    want = [i8.int8_gemm(*a) for a in args]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(i8.int8_gemm(*args[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i in range(2) for y in got[i])


def test_dispatched_route(cuda):
    x = _x(_gen(3), 5, 256, torch.float16)
    a, b = i8.quantize_int8(x), torch.ops.pi05_w4a4.quantize_int8(x)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    fn = torch.compile(lambda v: i8.int8_gemm(*i8.quantize_int8(v), a[0], a[1]), fullgraph=True, backend="eager")
    assert torch.equal(fn(x), i8.int8_gemm(*a, *a))

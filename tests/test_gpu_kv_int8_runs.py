"""Attention in several runs of pages at every head dimension, on two streams at once, and a captured append with all that
it writes.  References and tolerances are those of tests/test_gpu_kv_int8.py."""

from __future__ import annotations

import pytest
import torch
from test_gpu_kv_int8 import Cache, _check_attention, _gen, _i32, _kv, _pool

from pi05_fast.w4a4 import kv_int8 as kv

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("b,t,h,kvh,d,pages", [
    (1, 1, 8, 8, 64, 128), (4, 1, 32, 8, 64, 128), (4, 3, 6, 2, 64, 40), (1, 40, 4, 1, 64, 100), (1, 300, 8, 1, 64, 90),
    (1, 1, 8, 8, 128, 128), (4, 1, 32, 8, 128, 70), (4, 3, 6, 2, 128, 40), (1, 1, 8, 1, 256, 13), (4, 7, 8, 2, 256, 33),
])
def test_runs(cuda, b, t, h, kvh, d, pages, dtype):
    if torch.cuda.get_device_properties(0).multi_processor_count == 256:
        need = kv.load_int4_gemm().pi05w4a4_int8_kv_attention_workspace_bytes(b, t, h, kvh, d, pages)
        assert (need > 0) == ((t, pages) != (300, 90))  # those rows fill the CUs in one run
    gen = _gen(b + t + d + pages)
    cache, table = _pool(gen, b, pages, kvh, d)
    q = (torch.randn((b, t, h, d), device="cuda", generator=gen) * 1.5).to(dtype)
    lens = [pages * 64 - 5, 5, 0, pages * 32 + 1][:b]
    for causal in (True, False):
        _check_attention(q, cache, table, lens, d**-0.5, causal)


@pytest.mark.parametrize("d,pages", [(64, 30), (64, 128), (128, 30), (256, 30)])
def test_two_streams_of_their_own(cuda, d, pages):
    """Calls of one shape on two streams, each with its own queries, cache and lengths: a shared workspace would show."""
    gen = _gen(d)
    calls = []
    for lens in ([1900, 3, 700, 64], [5, 1800, 1900, 1]):
        cache, table = _pool(gen, 4, pages, 1, d)
        calls.append((torch.randn((4, 1, 8, d), device="cuda", generator=gen).half(), *cache, table, _i32(lens), 0.06))
    if torch.cuda.get_device_properties(0).multi_processor_count == 256:  # 30 pages of D = 64 are one run
        assert (kv.load_int4_gemm().pi05w4a4_int8_kv_attention_workspace_bytes(4, 1, 8, 1, d, pages) > 0) == ((d, pages) != (64, 30))
    want = [kv.int8_kv_attention(*c, return_lse=True) for c in calls]
    assert not torch.equal(want[0][0], want[1][0])
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(kv.int8_kv_attention(*calls[i], return_lse=True))
    torch.cuda.synchronize()
    assert all(torch.equal(a, want[i][0]) and torch.equal(s, want[i][1]) for i in range(2) for a, s in got[i])


def test_captured_append_writes_codes_and_scales(cuda):
    """Replays with moving lengths and growing values: all four tensors of the cache, against the eager call's."""
    gen = _gen(31)
    c = Cache(gen, 2, 3, 2, 128)
    eager = [t.clone() for t in c.t]
    k, v = _kv(gen, 2, 3, 2, 128, torch.float16)
    lens, counts = _i32([0, 0]), _i32([0, 0])
    kv.int8_kv_append(k, v, *c.t, c.table, lens, counts=counts)  # writes nothing
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv.int8_kv_append(k, v, *c.t, c.table, lens, counts=counts)
    for i in range(40):
        ki, vi = (x * (1 + i / 8) for x in _kv(gen, 2, 3, 2, 128, torch.float16))
        at, n = [3 * i, 2 * i], [3, 2]
        for dst, src in ((k, ki), (v, vi), (lens, _i32(at)), (counts, _i32(n))):
            dst.copy_(src)
        graph.replay()
        kv.int8_kv_append(ki, vi, *eager, c.table, _i32(at), counts=_i32(n))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(c.t, eager))

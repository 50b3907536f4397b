"""8-bit operators without a GPU: registration, fakes, refusals of the C ABI before any launch."""

from __future__ import annotations

import ctypes

import pytest
import torch

import pi05_fast.w4a4 as w4a4
from pi05_fast.w4a4 import extension as ext
from pi05_fast.w4a4 import int8 as i8
from pi05_fast.w4a4 import kv_int8 as kv

vp = ctypes.c_void_p
P = vp(4096)  # never dereferenced: the calls below are refused, or have nothing to do


@pytest.fixture(scope="module")
def lib():
    return ext.load_int4_gemm()


def _err(lib):
    return lib.pi05w4a4_last_error().decode()


def test_public_names_and_ops():
    for name in ("quantize_int8", "rms_norm_int8", "add_rms_norm_int8", "int8_gemm", "int8_kv_append",
                 "int8_kv_attention"):
        assert callable(getattr(w4a4, name)) and hasattr(torch.ops.pi05_w4a4, name)


def test_fakes_give_shapes_and_types():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x = torch.empty(2, 5, 256, dtype=torch.bfloat16)
        w = torch.empty(256, dtype=torch.bfloat16)
        q, s, h = i8.add_rms_norm_int8(x, x, w, 1e-6)
        assert (q.shape, q.dtype, s.shape, s.dtype, h.dtype) == (x.shape, torch.int8, x.shape[:2], torch.float32, x.dtype)
        q, s = i8.quantize_int8(x)
        y = i8.int8_gemm(q, s, torch.empty(33, 256, dtype=torch.int8), torch.empty(33), out_dtype=torch.bfloat16)
        assert tuple(y.shape) == (2, 5, 33) and y.dtype == torch.bfloat16
        kc, vc, ks, vs = kv.int8_kv_cache(4, 1, 64, "cpu")
        table, lens = torch.empty(2, 2, dtype=torch.int32), torch.empty(2, dtype=torch.int32)
        qq = torch.empty(2, 3, 4, 64, dtype=torch.float16)
        kv.int8_kv_append(qq[:, :, :1], qq[:, :, :1], kc, vc, ks, vs, table, lens)
        out, lse = kv.int8_kv_attention(qq, kc, vc, ks, vs, table, lens, 0.1, return_lse=True)
        assert out.shape == qq.shape and out.dtype == qq.dtype and tuple(lse.shape) == (2, 3, 4)


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 64, dtype=torch.float16)
    q = torch.zeros(2, 64, dtype=torch.int8)
    for call in (lambda: i8.quantize_int8(x), lambda: i8.rms_norm_int8(x, x[0], 1e-6),
                 lambda: i8.int8_gemm(q, torch.ones(2), q, torch.ones(2)),
                 lambda: kv.int8_kv_append(x[None, None], x[None, None], q, q, x, x, q, q),
                 lambda: kv.int8_kv_attention(x[None, None], q, q, x, x, q, q, 1.0)):
        with pytest.raises(RuntimeError, match="expects CUDA/HIP tensors"):
            call()
    with pytest.raises(RuntimeError, match="head_dim"):
        kv.int8_kv_cache(1, 1, 80, "cpu")


def _rows(lib, x=P, ldx=64, res=None, w=None, elem=0, m=2, k=64, q=P, scale=P, h=None):
    return lib.pi05w4a4_int8_rows(x, ldx, res, 64, w, 1e-6, 1, elem, m, k, q, scale, h, None)


@pytest.mark.parametrize("kw,text", [
    (dict(elem=2), "elem"), (dict(m=-1), "M must"), (dict(m=1 << 31), "M must"), (dict(k=12), "multiple of 8"),
    (dict(k=32776), "at most 32768"), (dict(k=0), "multiple of 8"), (dict(res=P), "norm weight"),
    (dict(res=P, w=P), "norm weight"), (dict(x=None), "null"), (dict(x=vp(4098)), "aligned"),
    (dict(ldx=60), "strides"), (dict(ldx=-8), "strides"), (dict(m=1 << 26), "one launch"),
    (dict(m=1 << 24, k=2056), "one launch"), (dict(m=1 << 22, k=8200), "one launch"),
])
def test_rows_refusals(lib, kw, text):
    assert _rows(lib, **kw) == 1 and text in _err(lib)
    assert _rows(lib, x=None, m=0) == 0


def _gemm(lib, q=P, ldq=64, m=2, k=64, w=P, ldw=64, n=8, elem=0, y=P, ws=None, wsb=0, res=None, ldr=8):
    return lib.pi05w4a4_int8_gemm(q, ldq, P, m, k, w, ldw, P, n, None, res, ldr, elem, y, ws, wsb, None)


@pytest.mark.parametrize("kw,text", [
    (dict(elem=-1), "elem"), (dict(m=-1), "M must"), (dict(n=-1), "N must"), (dict(n=(1 << 28) + 1), "N must"),
    (dict(k=72), "multiple of 16"), (dict(k=65552), "at most 65536"), (dict(q=None), "null"), (dict(q=vp(4104)), "aligned"),
    (dict(y=vp(4100)), "aligned"), (dict(ldq=72), "row strides"), (dict(ldw=(1 << 23) + 16), "row strides"),
    (dict(res=P, ldr=-1), "stride"), (dict(m=(1 << 31) - 1, n=1 << 28), "more tiles"),
])
def test_gemm_refusals(lib, kw, text):
    assert _gemm(lib, **kw) == 1 and text in _err(lib)
    assert _gemm(lib, q=None, m=0) == 0 and _gemm(lib, q=None, n=0) == 0


def test_gemm_workspace_is_checked(lib):
    need = lib.pi05w4a4_int8_gemm_workspace_bytes(1, 64, 16384)
    assert need > 0
    assert _gemm(lib, m=1, n=64, k=16384, ldq=16384, ldw=16384, ws=P, wsb=need - 4) == 3 and "workspace" in _err(lib)
    assert lib.pi05w4a4_int8_gemm_workspace_bytes(0, 64, 16384) == 0


I3 = ctypes.c_int64 * 3


def _append(lib, k=P, ks=I3(64, 64, 64), elem=0, b=1, t=1, kvh=1, d=64, kc=P, pages=1, table=P, tp=1, lens=P):
    return lib.pi05w4a4_int8_kv_append(k, ks, P, I3(64, 64, 64), elem, b, t, kvh, d, kc, P, P, P, pages, table, 1, tp,
                                       lens, None, None)


def _attend(lib, q=P, qs=I3(64, 64, 64), elem=0, b=1, t=1, h=1, kvh=1, d=64, kc=P, pages=1, table=P, tp=1, lens=P,
            scaling=1.0, out=P, ws=None, wsb=0):
    return lib.pi05w4a4_int8_kv_attention(q, qs, elem, b, t, h, kvh, d, kc, P, P, P, pages, table, 1, tp, lens, None,
                                          scaling, 1, out, None, ws, wsb, None)


_CACHE_REFUSALS = [
    (dict(elem=3), "elem"), (dict(d=80), "head_dim"), (dict(b=65536), "batch"), (dict(b=-1), "batch"), (dict(kvh=0), "KV heads"),
    (dict(pages=-1), "pages"), (dict(tp=-1), "table"), (dict(kc=None), "null"), (dict(lens=None), "null"),
    (dict(table=None), "null"), (dict(kc=vp(4104)), "aligned"),
]


@pytest.mark.parametrize("kw,text", _CACHE_REFUSALS + [
    (dict(k=vp(4104)), "aligned"), (dict(k=None), "null"), (dict(ks=I3(64, 60, 64)), "strides"), (dict(ks=I3(-8, 64, 64)), "strides"),
])
def test_append_refusals(lib, kw, text):
    assert _append(lib, **kw) == 1 and text in _err(lib)
    assert _append(lib, k=None, t=0) == 0 and _append(lib, k=None, b=0) == 0


@pytest.mark.parametrize("kw,text", _CACHE_REFUSALS + [
    (dict(q=vp(4104)), "aligned"), (dict(h=3, kvh=2), "multiple"), (dict(scaling=float("nan")), "finite"),
    (dict(out=None), "out must"), (dict(t=1 << 24, h=64), "at most 2^26"),
])
def test_attention_refusals(lib, kw, text):
    assert _attend(lib, **kw) == 1 and text in _err(lib)
    assert _attend(lib, q=None, t=0) == 0 and _attend(lib, q=None, b=0) == 0


def test_attention_workspace_is_checked(lib):
    need = lib.pi05w4a4_int8_kv_attention_workspace_bytes(1, 1, 8, 1, 256, 128)
    assert need > 0
    assert _attend(lib, h=8, d=256, tp=128, pages=128, ws=P, wsb=need - 4) == 3 and "workspace" in _err(lib)
    assert lib.pi05w4a4_int8_kv_attention_workspace_bytes(1, 1, 8, 1, 256, 0) == 0


@pytest.mark.parametrize("b,t,h,kvh,d,pages", [(1, 8320, 8, 1, 256, 2048), (1, 1, 8, 1, 256, 1 << 24), (3, 2000, 32, 8, 128, 4000),
                                               (65535, 1, 32767, 32767, 64, 1), (1, 1 << 24, 4, 1, 64, 1 << 24)])
def test_attention_workspace_is_bounded(lib, b, t, h, kvh, d, pages):
    assert lib.pi05w4a4_int8_kv_attention_workspace_bytes(b, t, h, kvh, d, pages) <= 1 << 28

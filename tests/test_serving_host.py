"""16-bit serving operators without a GPU: registration, fakes, refusals of the C ABI before any launch."""

from __future__ import annotations

import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fw

import pi05_fast.w4a4 as w4a4
from pi05_fast.w4a4 import extension as ext

vp = ctypes.c_void_p
P = vp(4096)  # never dereferenced: the calls below are refused, or have nothing to do
I3 = ctypes.c_int64 * 3
NAMES = ("qk_norm_rope", "qk_norm_rope_append", "kv_append", "kv_attention", "lora_add", "lora_add_")


@pytest.fixture(scope="module")
def lib():
    return ext.load_int4_gemm()


def _err(lib):
    return lib.pi05w4a4_last_error().decode()


def test_public_names_and_ops():
    for name in NAMES:
        assert callable(getattr(w4a4, name)) and hasattr(torch.ops.pi05_w4a4, name) and name in w4a4.__all__


def test_fakes_give_shapes_and_types():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        q, k = torch.empty(2, 3, 4, 64, dtype=torch.bfloat16), torch.empty(2, 3, 1, 64, dtype=torch.bfloat16)
        pos, freq = torch.empty(2, 3, dtype=torch.int32), torch.empty(32)
        a, b = w4a4.qk_norm_rope(q, k, None, None, 0.0, pos, freq, axes=[0] * 32)
        assert (a.shape, a.dtype, b.shape) == (q.shape, q.dtype, k.shape)
        cache = w4a4.kv_cache(4, 1, 64, torch.bfloat16, "cpu")
        table, lens = torch.empty(2, 2, dtype=torch.int32), torch.empty(2, dtype=torch.int32)
        w4a4.kv_append(k, k, *cache, table, lens)
        assert w4a4.qk_norm_rope_append(q, k, k, None, None, 0.0, pos, freq, *cache, table, lens).shape == q.shape
        out, lse = w4a4.kv_attention(q, *cache, table, lens, 0.1, return_lse=True)
        assert out.shape == q.shape and tuple(lse.shape) == (2, 3, 4) and lse.dtype == torch.float32
        y, x = torch.empty(5, 32, dtype=torch.float16), torch.empty(5, 64, dtype=torch.float16)
        la, lb = torch.empty(2, 16, 64, dtype=torch.float16), torch.empty(2, 32, 8, dtype=torch.float16)
        ids = torch.empty(5, dtype=torch.int32)
        assert w4a4.lora_add(y, x, la, lb, ids, slices=[16, 16]).shape == y.shape
        assert w4a4.lora_add_(y, x, la, lb, ids, slices=[16, 16]) is y


def _calls():
    q = torch.ones(1, 1, 1, 64, dtype=torch.float16)
    i, pos, freq = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32), torch.ones(32)
    cache = w4a4.kv_cache(1, 1, 64, torch.float16, "cpu")
    x, a, b = torch.ones(1, 64, dtype=torch.float16), torch.ones(1, 8, 64, dtype=torch.float16), torch.ones(1, 64, 8, dtype=torch.float16)
    return {
        "qk_norm_rope": lambda d: w4a4.qk_norm_rope(d(q), q, None, None, 0.0, pos, freq),
        "qk_norm_rope weight": lambda d: w4a4.qk_norm_rope(q, q, d(q[0, 0, 0].clone()), None, 0.0, pos, freq),
        "qk_norm_rope_append": lambda d: w4a4.qk_norm_rope_append(q, q, d(q), None, None, 0.0, pos, freq, *cache, i, i[0]),
        "kv_append": lambda d: w4a4.kv_append(d(q), q, *cache, i, i[0]),
        "kv_attention": lambda d: w4a4.kv_attention(d(q), *cache, i, i[0], 1.0),
        "lora_add": lambda d: w4a4.lora_add(x, d(x), a, b, i[0]),
        "lora_add_": lambda d: w4a4.lora_add_(d(x), x, a, b, i[0]),
        "op lora_add": lambda d: torch.ops.pi05_w4a4.lora_add(x, x, d(a), b, i[0], None, None),
        "op kv_attention": lambda d: torch.ops.pi05_w4a4.kv_attention(d(q), *cache, i, i[0], 1.0, True, None, False),
    }


@pytest.mark.parametrize("name", _calls())
def test_cpu_tensors_and_tangents_are_refused(name):
    call = _calls()[name]
    with pytest.raises(RuntimeError, match="expects CUDA/HIP tensors"):
        call(lambda t: t)
    with fw.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            call(lambda t: fw.make_dual(t, torch.ones_like(t)))


@pytest.mark.parametrize("name", ["qk_norm_rope_append", "kv_append", "lora_add_"])
def test_gradients_through_calls_in_place_are_refused(name):
    call = _calls()[name]
    with pytest.raises(RuntimeError, match="requires gradients"):
        call(lambda t: t.clone().requires_grad_())
    with torch.no_grad(), pytest.raises(RuntimeError, match="expects CUDA/HIP tensors"):
        call(lambda t: t.clone().requires_grad_())


def test_rope_axes():
    assert w4a4.rope_axes((2, 0, 3)) == (0, 0, 2, 2, 2)
    with pytest.raises(RuntimeError, match="head_dim"):
        w4a4.kv_cache(1, 1, 80, torch.float16, "cpu")
    with pytest.raises(RuntimeError, match="float16 or bfloat16"):
        w4a4.kv_cache(1, 1, 64, torch.float32, "cpu")


def _rope(lib, q=P, qs=I3(64, 64, 64), k=P, elem=0, b=1, t=1, h=1, kvh=1, d=64, qw=None, eps=1e-6, pos=P, ps=I3(0, 1, 1), pb=4, axes=1,
          amap=None, freq=P, rot=64, qo=P, ko=P):
    return lib.pi05w4a4_qk_norm_rope(q, qs, k, I3(64, 64, 64), elem, b, t, h, kvh, d, qw, None, eps, 1, pos, ps, pb, axes, amap, freq, rot,
                                     0, qo, ko, None)


def _rope_append(lib, q=P, qs=I3(64, 64, 64), k=P, v=P, elem=0, b=1, t=1, h=1, kvh=1, d=64, eps=1e-6, pos=P, ps=I3(0, 1, 1), pb=4, axes=1,
                 amap=None, freq=P, rot=64, qo=P, kc=P, pages=1, table=P, tp=1, lens=P, counts=None, qw=None):
    return lib.pi05w4a4_qk_norm_rope_append(q, qs, k, I3(64, 64, 64), v, I3(64, 64, 64), elem, b, t, h, kvh, d, qw, None, eps, 1, pos, ps, pb,
                                            axes, amap, freq, rot, 0, qo, kc, P, pages, table, 1, tp, lens, counts, None)


_ROPE_REFUSALS = [
    (dict(elem=2), "elem"), (dict(d=72), "head_dim"), (dict(d=528), "head_dim"), (dict(h=0), "positive"), (dict(kvh=0), "positive"),
    (dict(h=32768), "heads"), (dict(rot=8), "rotated"), (dict(rot=80), "rotated"), (dict(rot=-16), "rotated"), (dict(axes=0), "axes"),
    (dict(axes=5), "axes"), (dict(pb=2), "bytes"), (dict(eps=-1.0), "eps"), (dict(eps=float("inf")), "eps"), (dict(b=1 << 13, t=1 << 12), "2\\^24"),
    (dict(b=-1), "tokens"), (dict(amap=(ctypes.c_uint8 * 32)(*[1] * 32)), "axis 1 of 1"), (dict(q=None), "null"), (dict(q=vp(4104)), "aligned"),
    (dict(qs=I3(64, 60, 64)), "strides"), (dict(qs=I3(-8, 64, 64)), "strides"), (dict(qo=None), "outputs"), (dict(qw=vp(4104)), "norm weights"),
    (dict(pos=None), "null"), (dict(freq=None), "null"), (dict(pos=vp(4098)), "aligned"), (dict(pos=vp(4100), pb=8), "aligned"),
    (dict(ps=I3(0, -1, 1)), "positions"),
]


@pytest.mark.parametrize("kw,text", _ROPE_REFUSALS + [(dict(ko=None), "outputs")])
def test_rope_refusals(lib, kw, text):
    import re

    assert _rope(lib, **kw) == 1 and re.search(text, _err(lib))
    assert _rope(lib, q=None, t=0) == 0 and _rope(lib, q=None, b=0) == 0


_CACHE_REFUSALS = [
    (dict(elem=3), "elem"), (dict(d=80), "head_dim"), (dict(b=65536), "batch"), (dict(b=-1), "batch"), (dict(kvh=0), "KV heads"),
    (dict(pages=-1), "pages"), (dict(tp=-1), "table"), (dict(tp=(1 << 24) + 1), "table"), (dict(kc=None), "null"), (dict(lens=None), "null"),
    (dict(table=None), "null"), (dict(kc=vp(4104)), "aligned"),
]


@pytest.mark.parametrize("kw,text", _ROPE_REFUSALS + [(dict(v=None), "null"), (dict(v=vp(4104)), "aligned"), (dict(counts=vp(4098)), "counts"),
                                                      (dict(d=80, rot=16), "takes head_dim")] + _CACHE_REFUSALS[5:])
def test_rope_append_refusals(lib, kw, text):
    import re

    assert _rope_append(lib, **kw) == 1 and re.search(text, _err(lib))
    assert _rope_append(lib, q=None, t=0) == 0


def _append(lib, k=P, ks=I3(64, 64, 64), elem=0, b=1, t=1, kvh=1, d=64, kc=P, pages=1, table=P, tp=1, lens=P):
    return lib.pi05w4a4_kv_append(k, ks, P, I3(64, 64, 64), elem, b, t, kvh, d, kc, P, pages, table, 1, tp, lens, None, None)


def _attend(lib, q=P, qs=I3(64, 64, 64), elem=0, b=1, t=1, h=1, kvh=1, d=64, kc=P, pages=1, table=P, tp=1, lens=P, scaling=1.0, out=P, ws=None,
            wsb=0):
    return lib.pi05w4a4_kv_attention(q, qs, elem, b, t, h, kvh, d, kc, P, pages, table, 1, tp, lens, None, scaling, 1, out, None, ws, wsb, None)


@pytest.mark.parametrize("kw,text", _CACHE_REFUSALS + [
    (dict(k=vp(4104)), "aligned"), (dict(k=None), "null"), (dict(ks=I3(64, 60, 64)), "strides"), (dict(b=5000, t=5000), "2^24"),
])
def test_append_refusals(lib, kw, text):
    assert _append(lib, **kw) == 1 and text in _err(lib)
    assert _append(lib, k=None, t=0) == 0 and _append(lib, k=None, b=0) == 0


@pytest.mark.parametrize("kw,text", _CACHE_REFUSALS + [
    (dict(q=vp(4104)), "aligned"), (dict(h=3, kvh=2), "multiple"), (dict(scaling=float("nan")), "finite"), (dict(out=None), "out must"),
    (dict(t=1 << 24, h=64), "at most 2^26"),
])
def test_attention_refusals(lib, kw, text):
    assert _attend(lib, **kw) == 1 and text in _err(lib)
    assert _attend(lib, q=None, t=0) == 0 and _attend(lib, q=None, b=0) == 0


def test_new_tokens_are_apart_from_the_cache(lib):
    side = 2 * 64 * 64 * 2  # bytes of 2 pages of one head

    def append(k, v, kc, vc, pages=2, ks=I3(64, 64, 64), b=1, t=4):
        return lib.pi05w4a4_kv_append(vp(k), ks, vp(v), I3(64, 64, 64), 0, b, t, 1, 64, vp(kc), vp(vc), pages, P, 1, 1, P, None, None)

    at = 1 << 20
    for args in ((at, 1 << 16, at, 1 << 24), (at - 16, 1 << 16, at, 1 << 24), (1 << 16, at + side - 16, 1 << 24, at),
                 (1 << 16, at, at, 1 << 24)):
        assert append(*args) == 1 and "must not lie in the cache" in _err(lib)
    assert append(at - 4096, 1 << 16, at, 1 << 24, ks=I3(0, 1024, 64), t=4) == 1 and "must not lie in the cache" in _err(lib)
    for kc, vc in ((at, at), (at, at + side - 16), (at + 16, at)):
        assert append(1 << 10, 1 << 11, kc, vc) == 1 and "must not overlap" in _err(lib)


def test_adapters_of_too_many_rows(lib):
    far = vp(1 << 45)
    assert _lora(lib, x=far, m=1 << 26, per=1 << 26, n=1 << 12, ldy=1 << 12, ldo=1 << 12, ws=None, wsb=0) == 1
    assert "one launch" in _err(lib)
    assert _lora(lib, x=far, m=1 << 26, per=1 << 26, n=1 << 9, ldy=1 << 9, ldo=1 << 9, ws=None, wsb=0) == 3  # the workspace


def test_launches_of_too_many_waves(lib):
    big = dict(b=4096, t=4096, kvh=32767)
    assert _append(lib, **big) == 1 and "one launch" in _err(lib)
    assert _rope(lib, h=32767, **big) == 1 and "one launch" in _err(lib)
    assert _rope_append(lib, h=32767, **big) == 1 and "one launch" in _err(lib)


def test_attention_workspace_is_checked(lib):
    need = lib.pi05w4a4_kv_attention_workspace_bytes(1, 1, 8, 1, 256, 128)
    assert need > 0
    assert _attend(lib, h=8, d=256, tp=128, pages=128, ws=P, wsb=need - 4) == 3 and "workspace" in _err(lib)
    assert lib.pi05w4a4_kv_attention_workspace_bytes(1, 1, 8, 1, 256, 0) == 0


@pytest.mark.parametrize("b,t,h,kvh,d,pages", [(1, 8320, 8, 1, 256, 2048), (1, 1, 8, 1, 256, 1 << 24), (3, 2000, 32, 8, 128, 4000),
                                               (65535, 1, 32767, 32767, 64, 1), (1, 1 << 24, 4, 1, 64, 1 << 24)])
def test_attention_workspace_is_bounded(lib, b, t, h, kvh, d, pages):
    assert lib.pi05w4a4_kv_attention_workspace_bytes(b, t, h, kvh, d, pages) <= 1 << 28


def _lora(lib, y=P, ldy=32, x=vp(1 << 20), ldx=64, m=2, k=64, a=P, adapters=2, r=8, ids=P, per=1, n=32, slices=1, widths=None, elem=0, out=P, ldo=32,
          ws=P, wsb=1 << 30):
    return lib.pi05w4a4_lora_add(y, ldy, x, ldx, m, k, a, P, None, adapters, r, ids, per, n, slices, widths, elem, out, ldo, ws, wsb, None)


@pytest.mark.parametrize("kw,text", [
    (dict(elem=2), "elem"), (dict(m=-1), "M must"), (dict(m=(1 << 26) + 1), "M must"), (dict(per=0), "rows of an id"), (dict(k=12), "multiple of 8"),
    (dict(k=0), "multiple of 8"), (dict(k=(1 << 20) + 8), "at most 2^20"), (dict(n=-1), "N must"), (dict(n=(1 << 22) + 1), "N must"),
    (dict(r=4), "rank"), (dict(r=136), "rank"), (dict(slices=0), "slices"), (dict(slices=5), "slices"), (dict(adapters=-1), "adapters"),
    (dict(slices=2, widths=(ctypes.c_int32 * 2)(32, 0)), "has 0 columns"), (dict(slices=2, widths=(ctypes.c_int32 * 2)(16, 8)), "24 columns"),
    (dict(y=None), "null"), (dict(a=None), "null"), (dict(ids=None), "null"), (dict(x=vp(4104)), "aligned"), (dict(y=vp(4097)), "aligned"),
    (dict(ldx=60), "row stride of x"), (dict(ldo=31), "row strides"), (dict(ldy=-1), "row strides"),
    (dict(x=vp(4096 + 64), out=P), "must not overlap"), (dict(x=vp(8192), ldx=128, out=vp(8192 + 100), ldo=128), "must not overlap"),
    (dict(x=vp(8192 + 64), ldx=80, out=vp(8192), ldo=80), "must not overlap"),
])
def test_lora_refusals(lib, kw, text):
    assert _lora(lib, **kw) == 1 and text in _err(lib)
    assert _lora(lib, y=None, m=0) == 0 and _lora(lib, y=None, n=0) == 0


def test_lora_workspace_is_checked(lib):
    need = lib.pi05w4a4_lora_workspace_bytes(2, 1, 16384, 32, 8, 1, 2)
    assert need > 0 and need % (512 * 4) == 0
    assert _lora(lib, k=16384, ldx=16384, wsb=need - 4) == 3 and "workspace" in _err(lib)
    for args in ((0, 1, 64, 32, 8, 1, 2), (2, 1, 60, 32, 8, 1, 2), (2, 0, 64, 32, 8, 1, 2), (2, 1, 64, 0, 8, 1, 2), (2, 1, 64, 32, 8, 1, 0),
                 (2, 1, 64, 32, 8, 1, 2)):  # the last: one launch
        assert lib.pi05w4a4_lora_workspace_bytes(*args) == 0

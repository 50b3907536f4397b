"""Forward-mode duals and function transforms without a GPU: tangents are refused, by the wrappers and the dispatched
ops, and a transform takes the dispatched route."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fw

from pi05_fast.w4a4 import extension as ext
from pi05_fast.w4a4 import int8 as i8
from pi05_fast.w4a4 import kv_int8 as kv

X = torch.ones(4, 64, dtype=torch.float16)
Q = torch.ones(4, 64, dtype=torch.int8)
S = torch.ones(4)
I = torch.zeros(1, 1, dtype=torch.int32)
CACHE = kv.int8_kv_cache(1, 1, 64, "cpu")
PACKED = torch.zeros(16, 64 // 8 + 1, dtype=torch.int32)


def _heads(x):
    return x[:1].view(1, 1, 1, 64)


CALLS = {
    "quantize_int8": lambda d: i8.quantize_int8(d(X)),
    "rms_norm_int8": lambda d: i8.rms_norm_int8(X, d(X[0].clone()), 1e-6),
    "add_rms_norm_int8": lambda d: i8.add_rms_norm_int8(X, d(X), X[0].clone(), 1e-6),
    "int8_gemm scale": lambda d: i8.int8_gemm(Q, S, Q, d(S)),
    "int8_gemm residual": lambda d: i8.int8_gemm(Q, S, Q, S, residual=d(X[:, :4].contiguous())),
    "int8_kv_append": lambda d: kv.int8_kv_append(_heads(X), d(_heads(X)), *CACHE, I, I[0]),
    "int8_kv_attention": lambda d: kv.int8_kv_attention(d(_heads(X)), *CACHE, I, I[0], 1.0),
    "int4_gemm": lambda d: ext.int4_gemm(d(X), PACKED),
    "op quantize_int8": lambda d: torch.ops.pi05_w4a4.quantize_int8(d(X)),
    "op int8_gemm": lambda d: torch.ops.pi05_w4a4.int8_gemm(Q, d(S), Q, S, None, None, torch.float16),
    "op int8_kv_attention": lambda d: torch.ops.pi05_w4a4.int8_kv_attention(d(_heads(X)), *CACHE, I, I[0], 1.0, True, None, False),
}


@pytest.mark.parametrize("name", CALLS)
def test_tangents_are_refused(name):
    with fw.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            CALLS[name](lambda t: fw.make_dual(t, torch.ones_like(t)))
        # inside a level, without a tangent: as ever (no CPU form)
        with pytest.raises(RuntimeError, match="expects CUDA/HIP tensors"):
            CALLS[name](lambda t: t)


def test_jvp_is_refused():
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(lambda s: i8.int8_gemm(Q, S, Q, s), (S,), (S,))


def test_transforms_take_the_dispatched_route():
    seen = []

    def fn(x):
        seen.append(ext._direct(x))
        return x

    assert ext._direct(X)
    torch.vmap(fn)(X)
    torch.func.functionalize(fn)(X)
    assert seen == [False, False] and ext._direct(X)
    with pytest.raises(RuntimeError, match="expects CUDA/HIP tensors"):
        torch.vmap(lambda x: i8.quantize_int8(x)[1])(X[:, None])

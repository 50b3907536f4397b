"""8-bit rows and products: the W8A8 counterpart of the INT4 ops, for layers that 4 bits hurt.

* ``quantize_int8``, ``rms_norm_int8``, ``add_rms_norm_int8``: rows to int8 codes with one fp32
  scale each, as they are, behind an RMSNorm, or behind a residual add and an RMSNorm (which
  returns the new residual stream too), in one kernel;
* ``int8_gemm``: codes x int8 weights with token and channel scales, and a bias and a residual in
  the epilogue.

Weights need no layout of their own: ``quantize_int8(w)`` of an ``nn.Linear`` weight [N, K] gives
its codes and channel scales.  The reference has no 8-bit path; the ops are registered beside
its own as ``torch.ops.pi05_w4a4.*`` with shape-only fakes, and there is no CPU fallback.
"""

from __future__ import annotations

import torch

from pi05_fast.w4a4 import extension as _ext
from pi05_fast.w4a4.extension import (_check, _direct, _on_device, _ptr, _refuse_tangents, _stream, _workspace,
                                      load_int4_gemm)

ELEM = {torch.float16: 0, torch.bfloat16: 1}
MAX_ROW = 32768  # longest row of the quantizers
MAX_K = 65536  # longest K of the product: its int32 sums are exact
MAX_N = 1 << 28  # most weight rows of the product

_GEMM_WS: dict[tuple, int] = {}


def _rows(x: torch.Tensor, k: int, name: str) -> tuple[torch.Tensor, int]:
    """x as rows of k contiguous elements at one stride (a multiple of 8 elements, 16-byte
    aligned), copied only where it is not that already: (tensor, row stride)."""
    if x.is_contiguous():
        ld = k
    elif x.dim() == 2 and x.stride(1) == 1 and x.stride(0) % 8 == 0:
        ld = x.stride(0)
    else:
        x, ld = x.contiguous(), k
    if x.data_ptr() % 16:
        x, ld = x.clone(memory_format=torch.contiguous_format), k
    return x, ld


def _quantize_impl(x, residual, weight, eps, unit_offset, what):
    if not x.is_cuda:
        raise RuntimeError(f"{what} expects CUDA/HIP tensors")
    elem = ELEM.get(x.dtype)
    if elem is None:
        raise RuntimeError(f"{what} takes float16 or bfloat16, got {x.dtype}")
    if x.dim() == 0 or x.size(-1) <= 0:
        raise RuntimeError(f"{what} expects rows of at least one element")
    k = int(x.size(-1))
    if k % 8 or k > MAX_ROW:
        raise RuntimeError(f"{what}: K must be a multiple of 8 of at most {MAX_ROW}, got {k}")
    dev, shape = x.device, x.shape
    ldr = 0
    if weight is not None:
        if weight.device != dev or weight.dtype != x.dtype or weight.dim() != 1 or int(weight.numel()) != k:
            raise RuntimeError(f"{what}: the norm weight must be a {x.dtype} tensor [{k}] on {dev}")
        if not weight.is_contiguous() or weight.data_ptr() % 16:
            weight = weight.clone(memory_format=torch.contiguous_format)
    if residual is not None:
        if residual.device != dev or residual.dtype != x.dtype or residual.shape != shape:
            raise RuntimeError(f"{what}: the residual must be a {x.dtype} tensor {tuple(shape)} on {dev}")
        residual, ldr = _rows(residual, k, "residual")
    xr, ldx = _rows(x, k, "x")
    m = x.numel() // k
    q = torch.empty_like(x, dtype=torch.int8, memory_format=torch.contiguous_format)
    scale = torch.empty(shape[:-1], dtype=torch.float32, device=dev)
    h = torch.empty_like(x, memory_format=torch.contiguous_format) if residual is not None else None
    lib = _ext._lib if _ext._lib is not None else load_int4_gemm()
    with _on_device(dev):
        _check(lib.pi05w4a4_int8_rows(xr.data_ptr(), ldx, _ptr(residual), ldr, _ptr(weight), eps,
                                      1 if unit_offset else 0, elem, m, k, q.data_ptr(), scale.data_ptr(), _ptr(h),
                                      _stream(dev)), "pi05w4a4_int8_rows")
    return q, scale, h


def _matrix(t: torch.Tensor, k: int) -> tuple[torch.Tensor, int]:
    """An int8 operand as rows of k bytes at one stride (a multiple of 16), copied where it is not that."""
    if t.is_contiguous():
        ld = k
    elif t.dim() == 2 and t.stride(1) == 1 and t.stride(0) % 16 == 0 and t.stride(0) <= 1 << 23:
        ld = t.stride(0)
    else:
        t, ld = t.contiguous(), k
    if t.data_ptr() % 16:
        t, ld = t.clone(memory_format=torch.contiguous_format), k
    return t, ld


def _gemm_impl(q, q_scale, w, w_scale, bias, residual, out_dtype):
    if not q.is_cuda:
        raise RuntimeError("int8_gemm expects CUDA/HIP tensors")
    dev = q.device
    elem = ELEM.get(out_dtype)
    if elem is None:
        raise RuntimeError(f"int8_gemm writes float16 or bfloat16, got {out_dtype}")
    if q.dtype != torch.int8 or w.dtype != torch.int8 or w.dim() != 2 or q.dim() == 0:
        raise RuntimeError("int8_gemm takes int8 codes [..., K] and int8 weights [N, K]")
    k, n = int(q.size(-1)), int(w.size(0))
    if int(w.size(1)) != k:
        raise RuntimeError(f"int8_gemm: the codes have K={k}, the weights {tuple(w.shape)}")
    if k <= 0 or k % 16 or k > MAX_K:
        raise RuntimeError(f"int8_gemm: K must be a multiple of 16 of at most {MAX_K}, got {k}")
    if n > MAX_N:  # here: the library takes N as 32 bits
        raise RuntimeError(f"int8_gemm: N must be at most {MAX_N}, got {n}")
    lead = q.shape[:-1]
    shape = (*lead, n)
    m = q.numel() // k
    if q_scale.dtype != torch.float32 or q_scale.device != dev or q_scale.shape != lead:
        raise RuntimeError(f"int8_gemm: q_scale must be float32 {tuple(lead)} on {dev}, got {q_scale.dtype} "
                           f"{tuple(q_scale.shape)} on {q_scale.device}")
    if w_scale.dtype != torch.float32 or w_scale.device != dev or w_scale.shape != (n,):
        raise RuntimeError(f"int8_gemm: w_scale must be float32 [{n}] on {dev}, got {w_scale.dtype} "
                           f"{tuple(w_scale.shape)} on {w_scale.device}")
    if w.device != dev:
        raise RuntimeError(f"int8_gemm: the weights must be on {dev}, got {w.device}")
    if bias is not None:
        if bias.device != dev or bias.dtype != out_dtype or bias.dim() != 1 or int(bias.numel()) != n:
            raise RuntimeError(f"int8_gemm: the bias must be a {out_dtype} tensor [{n}] on {dev}")
        bias = bias.contiguous()
    ldr = 0
    if residual is not None:
        if residual.device != dev or residual.dtype != out_dtype or residual.shape != shape:
            raise RuntimeError(f"int8_gemm: the residual must be a {out_dtype} tensor {tuple(shape)} on {dev}")
        if residual.is_contiguous():
            ldr = n
        elif residual.dim() == 2 and residual.stride(1) == 1:
            ldr = residual.stride(0)
        else:
            residual, ldr = residual.contiguous(), n
    q, ldq = _matrix(q, k)
    w, ldw = _matrix(w, k)
    q_scale, w_scale = q_scale.contiguous(), w_scale.contiguous()
    y = torch.empty(shape, dtype=out_dtype, device=dev)
    lib = _ext._lib if _ext._lib is not None else load_int4_gemm()
    with _on_device(dev):
        key = (dev.index, m, n, k)
        need = _GEMM_WS.get(key)
        if need is None:
            if len(_GEMM_WS) > 4096:
                _GEMM_WS.clear()
            need = _GEMM_WS[key] = int(lib.pi05w4a4_int8_gemm_workspace_bytes(m, n, k))
        ws = _workspace(dev, need) if need else None
        _check(lib.pi05w4a4_int8_gemm(q.data_ptr(), ldq, q_scale.data_ptr(), m, k, w.data_ptr(), ldw,
                                      w_scale.data_ptr(), n, _ptr(bias), _ptr(residual), ldr, elem, y.data_ptr(),
                                      _ptr(ws), need, _stream(dev)), "pi05w4a4_int8_gemm")
    return y


# ----------------------------------------------------------------------------- custom ops
@torch.library.custom_op("pi05_w4a4::quantize_int8", mutates_args=())
def _quantize_op(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    _refuse_tangents(x)
    return _quantize_impl(x, None, None, 0.0, False, "quantize_int8")[:2]


def _fake_rows(x):
    return x.new_empty(x.shape, dtype=torch.int8), x.new_empty(x.shape[:-1], dtype=torch.float32)


@_quantize_op.register_fake
def _quantize_fake(x):
    return _fake_rows(x)


@torch.library.custom_op("pi05_w4a4::rms_norm_int8", mutates_args=())
def _rms_norm_op(x: torch.Tensor, weight: torch.Tensor, eps: float,
                 unit_offset: bool) -> tuple[torch.Tensor, torch.Tensor]:
    _refuse_tangents(x, weight)
    return _quantize_impl(x, None, weight, eps, unit_offset, "rms_norm_int8")[:2]


@_rms_norm_op.register_fake
def _rms_norm_fake(x, weight, eps, unit_offset):
    return _fake_rows(x)


@torch.library.custom_op("pi05_w4a4::add_rms_norm_int8", mutates_args=())
def _add_rms_norm_op(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, eps: float,
                     unit_offset: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    _refuse_tangents(x, residual, weight)
    return _quantize_impl(x, residual, weight, eps, unit_offset, "add_rms_norm_int8")


@_add_rms_norm_op.register_fake
def _add_rms_norm_fake(x, residual, weight, eps, unit_offset):
    return (*_fake_rows(x), x.new_empty(x.shape))


@torch.library.custom_op("pi05_w4a4::int8_gemm", mutates_args=())
def _gemm_op(q: torch.Tensor, q_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
             bias: torch.Tensor | None, residual: torch.Tensor | None, out_dtype: torch.dtype) -> torch.Tensor:
    _refuse_tangents(q_scale, w_scale, bias, residual)
    return _gemm_impl(q, q_scale, w, w_scale, bias, residual, out_dtype)


@_gemm_op.register_fake
def _gemm_fake(q, q_scale, w, w_scale, bias, residual, out_dtype):
    return q.new_empty((*q.shape[:-1], w.shape[0]), dtype=out_dtype)


# ----------------------------------------------------------------------------- public functions
def quantize_int8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows of x (fp16 or bf16 [..., K], K % 8 == 0, K <= 32768) to int8 codes [..., K] and
    fp32 scales [...]: scale = max|row| / 127 + 1e-12, code = rint(x / scale).  A row that
    holds a NaN or an infinity gets the scale NaN and codes 0.  Also a Linear's weight
    [N, K] to its codes and channel scales."""
    if _direct(x):
        return _quantize_impl(x, None, None, 0.0, False, "quantize_int8")[:2]
    return torch.ops.pi05_w4a4.quantize_int8(x)


def rms_norm_int8(x: torch.Tensor, weight: torch.Tensor, eps: float,
                  unit_offset: bool = True) -> tuple[torch.Tensor, torch.Tensor]:
    """``quantize_int8`` of the RMSNorm of x, x / sqrt(mean(x^2) + eps) * (unit_offset + weight),
    held in fp32 between the two (``rms_norm`` would round it to 16 bits).  Squares past fp32's
    range do no harm; a row that holds a NaN or an infinity, or is past fp32 behind the norm,
    gets the scale NaN and codes 0."""
    if _direct(x, weight):
        return _quantize_impl(x, None, weight, float(eps), bool(unit_offset), "rms_norm_int8")[:2]
    return torch.ops.pi05_w4a4.rms_norm_int8(x, weight, float(eps), bool(unit_offset))


def add_rms_norm_int8(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, eps: float,
                      unit_offset: bool = True) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(codes, scales, h): h = x + residual in their type (the new residual stream) and
    ``rms_norm_int8`` of h, in one pass."""
    if _direct(x, residual, weight):
        return _quantize_impl(x, residual, weight, float(eps), bool(unit_offset), "add_rms_norm_int8")
    return torch.ops.pi05_w4a4.add_rms_norm_int8(x, residual, weight, float(eps), bool(unit_offset))


def int8_gemm(q: torch.Tensor, q_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
              bias: torch.Tensor | None = None, residual: torch.Tensor | None = None,
              out_dtype: torch.dtype = torch.float16) -> torch.Tensor:
    """(q w^T) * q_scale * w_scale + bias + residual: int8 codes q [..., K] with fp32 scales
    [...], int8 weights w [N, K] with fp32 scales [N] (K % 16 == 0, K <= 65536; any N), bias
    [N] and residual [..., N] in ``out_dtype`` (fp16 or bf16).  The integer sums are exact,
    the epilogue is fp32 with one rounding."""
    if _direct(q, q_scale, w, w_scale, bias, residual):
        return _gemm_impl(q, q_scale, w, w_scale, bias, residual, out_dtype)
    return torch.ops.pi05_w4a4.int8_gemm(q, q_scale, w, w_scale, bias, residual, out_dtype)

"""Low-rank adapters of many requests beside a shared projection.

``lora_add(y, x, a, b, ids, scale)`` adds scale[id] (x A[id]^T) B[id]^T to the output y of a projection of x
(``int4_gemm``, ``int8_gemm`` or any other), each row with the adapter of its request.  Rows need no
order: a batch of decoded tokens may have an adapter each, a prompt one, and rows without one keep y.
"""

from __future__ import annotations

import ctypes
from collections.abc import Sequence

import torch

from pi05_fast.w4a4 import extension as _ext
from pi05_fast.w4a4.extension import (_changed, _check, _direct, _on_device, _ptr, _refuse_gradients, _refuse_tangents, _stream,
                                      _workspace, load_int4_gemm)
from pi05_fast.w4a4.int8 import ELEM
from pi05_fast.w4a4.rope import _meta, _plan

MAX_RANK = 128
MAX_SLICES = 4
MAX_ROWS = 1 << 26
MAX_K = 1 << 20
MAX_N = 1 << 22


def _row_stride(t: torch.Tensor) -> int | None:
    """The one stride at which the rows of t [..., K] lie, or None."""
    if t.dim() < 1 or (t.stride(-1) != 1 and t.size(-1) > 1):
        return None
    if t.is_contiguous():
        return t.size(-1)
    ld = span = None
    for size, stride in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        if size == 1:
            continue
        if ld is None:
            ld, span = stride, stride * size
        elif stride != span:
            return None
        else:
            span *= size
    return t.size(-1) if ld is None else ld


def _may_share(x: torch.Tensor, y: torch.Tensor) -> bool:
    """Whether x and y can hold the same bytes: x is then copied, as the kernels read it while they write y."""
    if x.data_ptr() == y.data_ptr():
        return True
    ends = []
    for t in (x, y):
        ends.append(t.data_ptr() + 2 * (1 + sum((n - 1) * st for n, st in zip(t.shape, t.stride()))))
    return x.data_ptr() < ends[1] and y.data_ptr() < ends[0]


def _check_lora(what, y, x, a, b, ids, scale, widths, in_place):
    """The checks, and what they find: (m, k, n, r, adapters, rows an id), the row strides of y and x (None: to be copied), the widths
    for the library and the workspace."""
    if not y.is_cuda:
        raise RuntimeError(f"{what} expects CUDA/HIP tensors")
    dev, dtype = y.device, y.dtype
    elem = ELEM.get(dtype)
    if elem is None or x.dtype != dtype or a.dtype != dtype or b.dtype != dtype:
        raise RuntimeError(f"{what} takes float16 or bfloat16 tensors of one type, got y {dtype}, x {x.dtype}, a {a.dtype}, b {b.dtype}")
    if y.dim() < 1 or x.dim() != y.dim() or x.shape[:-1] != y.shape[:-1]:
        raise RuntimeError(f"{what} expects y [..., N] and x [..., K] of the same rows, got {tuple(y.shape)} and {tuple(x.shape)}")
    lead, n, k = y.shape[:-1], y.size(-1), x.size(-1)
    widths = (n,) if widths is None else widths
    if not 1 <= len(widths) <= MAX_SLICES or sum(widths) != n or (n > 0 and min(widths) <= 0):
        raise RuntimeError(f"{what}: slices are 1 to {MAX_SLICES} positive widths whose sum is N = {n}, got {widths}")
    if a.dim() != 3 or b.dim() != 3 or a.size(0) != b.size(0) or a.size(2) != k or b.size(1) != n \
            or a.size(1) != len(widths) * b.size(2):
        raise RuntimeError(f"{what} expects a [adapters, {len(widths)} * R, {k}] and b [adapters, {n}, R], got {tuple(a.shape)} and "
                           f"{tuple(b.shape)}")
    adapters, r = a.size(0), b.size(2)
    if k <= 0 or k % 8 or k > MAX_K or r <= 0 or r % 8 or r > MAX_RANK or n > MAX_N or adapters > 0x7fffffff:
        raise RuntimeError(f"{what}: K and the rank must be multiples of 8 of at most {MAX_K} and {MAX_RANK} and N at most {MAX_N}, "
                           f"got K={k}, rank {r}, N={n}")
    if ids.dtype != torch.int32 or ids.dim() > len(lead) or ids.shape != lead[:ids.dim()]:
        raise RuntimeError(f"{what}: ids must be int32 of the first dimensions of {tuple(lead)}, got {ids.dtype} {tuple(ids.shape)}")
    if scale is not None and (scale.dtype != torch.float32 or scale.shape != (adapters,)):
        raise RuntimeError(f"{what}: scale must be float32 [{adapters}], got {scale.dtype} {tuple(scale.shape)}")
    for t in (x, a, b, ids, scale):
        if t is not None and t.device != dev:
            raise RuntimeError(f"{what}: all tensors must be on {dev}, got {t.device}")
    m = 1
    for size in lead:
        m *= size
    if m > MAX_ROWS:
        raise RuntimeError(f"{what}: at most {MAX_ROWS} rows, got {m}")
    ldy, ldx = _row_stride(y), _row_stride(x)
    if in_place and (ldy is None or (m > 1 and ldy < n)):
        raise RuntimeError(f"{what}: the rows of y must lie at one stride and apart, got strides {y.stride()} of {tuple(y.shape)}")
    per_id = m // ids.numel() if m > 0 else 1
    need = 0
    if m > 0 and n > 0:
        with _on_device(dev):
            need = int(load_int4_gemm().pi05w4a4_lora_workspace_bytes(m, per_id, k, n, r, len(widths), adapters))
    return ((m, k, n, r, adapters, per_id), ldy, None if ldx is None or ldx % 8 else ldx,
            (ctypes.c_int32 * len(widths))(*widths), elem, need)


def _lora_impl(y, x, a, b, ids, scale, slices, in_place):
    what = "lora_add_" if in_place else "lora_add"
    slices = None if slices is None else tuple(slices)
    (m, k, n, r, adapters, per_id), ldy, ldx, widths, elem, need = _plan(
        (what, slices, y.dtype, y.device, y.shape, y.stride(), x.dtype, x.device, x.shape, x.stride(), a.dtype, a.device, a.shape, b.dtype,
         b.device, b.shape, ids.dtype, ids.device, ids.shape, _meta(scale)),
        lambda: _check_lora(what, y, x, a, b, ids, scale, slices, in_place))
    dev = y.device
    if in_place:
        out, ldo = y, max(ldy, n)  # of a single row the stride may be anything
    else:
        out, ldo = torch.empty_like(y, memory_format=torch.contiguous_format), n
        if ldy is None:
            y, ldy = y.contiguous(), n
    if m == 0 or n == 0:
        return out
    if ldx is None or x.data_ptr() % 16 or (in_place and _may_share(x, y)):
        x, ldx = x.clone(memory_format=torch.contiguous_format), k
    a, b, ids = _whole(a), _whole(b), ids.contiguous()
    scale = None if scale is None else scale.contiguous()
    lib = _ext._lib if _ext._lib is not None else load_int4_gemm()
    with _on_device(dev):
        ws = _workspace(dev, need) if need else None
        _check(lib.pi05w4a4_lora_add(y.data_ptr(), ldo if in_place else ldy, x.data_ptr(), ldx, m, k, a.data_ptr(), b.data_ptr(),
                                     _ptr(scale), adapters, r, ids.data_ptr(), per_id, n, len(widths), widths, elem, out.data_ptr(),
                                     ldo, _ptr(ws), need, _stream(dev)), "pi05w4a4_lora_add")
    return out


def _whole(t: torch.Tensor) -> torch.Tensor:
    if t.is_contiguous() and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


# ----------------------------------------------------------------------------- custom ops
@torch.library.custom_op("pi05_w4a4::lora_add", mutates_args=())
def _lora_op(y: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, ids: torch.Tensor,
             scale: torch.Tensor | None, slices: Sequence[int] | None) -> torch.Tensor:
    _refuse_tangents(y, x, a, b, scale)
    return _lora_impl(y, x, a, b, ids, scale, slices, False)


@_lora_op.register_fake
def _lora_fake(y, x, a, b, ids, scale, slices):
    return y.new_empty(y.shape)


@torch.library.custom_op("pi05_w4a4::lora_add_", mutates_args=("y",))
def _lora_inplace_op(y: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, ids: torch.Tensor,
                     scale: torch.Tensor | None, slices: Sequence[int] | None) -> None:
    _refuse_tangents(y, x, a, b, scale)
    _lora_impl(y, x, a, b, ids, scale, slices, True)


@_lora_inplace_op.register_fake
def _lora_inplace_fake(y, x, a, b, ids, scale, slices):
    return None


# ----------------------------------------------------------------------------- public functions
def lora_add(y: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, ids: torch.Tensor,
             scale: torch.Tensor | None = None, slices: Sequence[int] | None = None) -> torch.Tensor:
    """y + scale[id] * (x a[id]^T) b[id]^T, a new tensor: y [..., N] and x [..., K] (fp16 or bf16, K a multiple of
    8), a [adapters, R, K], b [adapters, N, R] (R a multiple of 8 of at most 128; smaller ranks are
    padded with zeros), ids int32 of the first dimensions of the rows ([B] for one adapter a request, or
    one for each row), scale fp32 [adapters] (None: 1).  Ids outside [0, adapters) name no adapter: those
    rows are y.  Sums are fp32, with one rounding; the first one's enter the second product to 2^-22 in fp16, whole in bf16.

    ``slices`` (up to four widths, their sum N) are the parts of a joined projection, which have first
    factors of their own: a is then [adapters, len(slices) * R, K], part g's rows g R .. g R + R - 1, and
    columns of part g take the R sums of that part.  There are no derivatives."""
    if _direct(y, x, a, b, ids, scale):
        return _lora_impl(y, x, a, b, ids, scale, slices, False)
    return torch.ops.pi05_w4a4.lora_add(y, x, a, b, ids, scale, None if slices is None else list(slices))


def lora_add_(y: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, ids: torch.Tensor,
              scale: torch.Tensor | None = None, slices: Sequence[int] | None = None) -> torch.Tensor:
    """``lora_add`` into y, which may be a part of a wider output (rows at one stride), and y.  Rows without an
    adapter are not touched.  An x in the same memory is copied first.  Arguments that require gradients are refused."""
    if _direct(y, x, a, b, ids, scale):
        _lora_impl(y, x, a, b, ids, scale, slices, True)
        _changed(y)
        return y
    _refuse_gradients("lora_add_", y, x, a, b, scale)
    torch.ops.pi05_w4a4.lora_add_(y, x, a, b, ids, scale, None if slices is None else list(slices))
    return y

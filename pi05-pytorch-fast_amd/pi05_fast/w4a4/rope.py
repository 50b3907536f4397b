"""Norm and rotation of query and key heads between a joined QKV product and the attention.

``qk_norm_rope``: an RMSNorm of each query and key head (or none) and the rotation by position in one
pass, for one position a token or several (time, height and width of images and video), and
for heads of which a part is rotated.  ``kv.qk_norm_rope_append`` does the same on the way into a KV
cache.  The fused prefix path (``prefix_attention``, ``rms_norm_int4_gemm3_rope``) rotates inside its
own kernels, by tables of one position and without a head norm.
"""

from __future__ import annotations

import ctypes
from collections.abc import Sequence

import torch

from pi05_fast.w4a4 import extension as _ext
from pi05_fast.w4a4.extension import _check, _direct, _on_device, _ptr, _refuse_tangents, _stream, load_int4_gemm
from pi05_fast.w4a4.int8 import ELEM

MAX_HEAD_DIM = 512
MAX_AXES = 4
MAX_HEADS = 32767
MAX_TOKENS = 1 << 24  # tokens of a call

# What the checks of a call find depends on its tensors' types, devices, shapes and strides only: the arguments of
# calls that passed them, by these (one flat tuple, written out at each call: half the time of a tuple of tuples).
_PLANS: dict[tuple, tuple] = {}


def _meta(t: torch.Tensor | None):
    return None if t is None else (t.dtype, t.device, t.shape, t.stride())


def _strides(t: torch.Tensor):
    """The first three strides of t [B, T, heads, D] for the library, or None where its rows have to be copied
    (16-byte alignment of the first is not looked at)."""
    st, sz = t.stride(), t.shape
    key = tuple(0 if sz[i] == 1 else st[i] for i in range(3))
    if st[3] != 1 or key[0] % 8 or key[1] % 8 or key[2] % 8:
        return None
    return (ctypes.c_int64 * 3)(*key)


def _heads(t: torch.Tensor, strides) -> tuple[torch.Tensor, ctypes.Array]:
    """t with rows that the library takes, copied only where it has none."""
    if strides is None or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
        strides = (ctypes.c_int64 * 3)(*t.stride()[:3])
    return t, strides


def _axis_map(what, axes, pairs: int, count: int):
    """The axis of each pair as bytes for the library (None: all on the first)."""
    if axes is None:
        if count > 1:
            raise RuntimeError(f"{what}: positions of {count} axes need `axes`, the axis of each of the {pairs} rotated pairs")
        return None
    if len(axes) != pairs:
        raise RuntimeError(f"{what}: axes must name the axis of each of the {pairs} rotated pairs, got {len(axes)}")
    if any(not 0 <= a < count for a in axes):
        raise RuntimeError(f"{what}: axes must be in [0, {count}), the positions' axes, got {sorted(set(axes))}")
    return (ctypes.c_uint8 * pairs)(*axes)


def _check_weight(what, name, w, x, d):
    if w is not None and (w.device != x.device or w.dtype != x.dtype or w.shape != (d,)):
        raise RuntimeError(f"{what}: {name} must be a {x.dtype} tensor [{d}] on {x.device}")


def _weight(w: torch.Tensor | None) -> torch.Tensor | None:
    if w is not None and (not w.is_contiguous() or w.data_ptr() % 16):
        w = w.clone(memory_format=torch.contiguous_format)
    return w


def _check_rope(what, q, k, q_weight, k_weight, positions, inv_freq, axes):
    """The checks shared by the forms of the call, and what they find: (elem, b, t, h, kvh, d), the strides of q, k and the
    positions and their bytes, the number of axes and their map, the rotated dimensions."""
    if not q.is_cuda:
        raise RuntimeError(f"{what} expects CUDA/HIP tensors")
    dev = q.device
    elem = ELEM.get(q.dtype)
    if elem is None or k.dtype != q.dtype:
        raise RuntimeError(f"{what} takes float16 or bfloat16 queries and keys of one type, got {q.dtype} and {k.dtype}")
    if q.dim() != 4 or k.dim() != 4 or k.shape[:2] != q.shape[:2] or k.size(3) != q.size(3) or k.device != dev:
        raise RuntimeError(f"{what} expects q [B, T, H, D] and k [B, T, KVH, D] on one device, got {tuple(q.shape)} and "
                           f"{tuple(k.shape)}")
    b, t, h, d = q.shape
    kvh = k.size(2)
    if d % 16 or not 0 < d <= MAX_HEAD_DIM:
        raise RuntimeError(f"{what}: head_dim must be a multiple of 16 of at most {MAX_HEAD_DIM}, got {d}")
    if not 0 < h <= MAX_HEADS or not 0 < kvh <= MAX_HEADS or b * t > MAX_TOKENS:  # here: the library takes them as 32 bits
        raise RuntimeError(f"{what}: 1 to {MAX_HEADS} heads and at most {MAX_TOKENS} tokens, got {h} and {kvh} heads, {b} x {t}")
    _check_weight(what, "q_weight", q_weight, q, d)
    _check_weight(what, "k_weight", k_weight, q, d)
    if inv_freq.dtype != torch.float32 or inv_freq.dim() != 1 or inv_freq.device != dev:
        raise RuntimeError(f"{what}: inv_freq must be float32 [rotated dimensions / 2] on {dev}, got {inv_freq.dtype} "
                           f"{tuple(inv_freq.shape)} on {inv_freq.device}")
    pairs = inv_freq.numel()
    if pairs % 8 or 2 * pairs > d:
        raise RuntimeError(f"{what}: the rotated dimensions must be a multiple of 16 of at most {d}, got {2 * pairs}")
    if positions.dtype not in (torch.int32, torch.int64) or positions.device != dev or positions.dim() not in (2, 3) \
            or positions.shape[-2:] != (b, t) or (positions.dim() == 3 and not 1 <= positions.size(0) <= MAX_AXES):
        raise RuntimeError(f"{what}: positions must be int32 or int64 [{b}, {t}], or [axes, {b}, {t}] of at most {MAX_AXES} "
                           f"axes, on {dev}, got {positions.dtype} {tuple(positions.shape)} on {positions.device}")
    count = positions.size(0) if positions.dim() == 3 else 1
    amap = _axis_map(what, axes, pairs, count)
    ps = positions.stride() if positions.dim() == 3 else (0, *positions.stride())
    return ((elem, b, t, h, kvh, d), _strides(q), _strides(k), (ctypes.c_int64 * 3)(*ps), positions.element_size(), count, amap,
            2 * pairs)


def _plan(key: tuple, make) -> tuple:
    got = _PLANS.get(key)
    if got is None:
        got = make()
        if len(_PLANS) > 4096:
            _PLANS.clear()
        _PLANS[key] = got
    return got


def _rope_impl(q, k, q_weight, k_weight, eps, positions, inv_freq, unit_offset, interleaved, axes):
    what = "qk_norm_rope"
    axes = None if axes is None else tuple(axes)
    shape, qs, ks, ps, pos_bytes, count, amap, rot = _plan(
        (what, axes, q.dtype, q.device, q.shape, q.stride(), k.dtype, k.device, k.shape, k.stride(), _meta(q_weight), _meta(k_weight),
         positions.dtype, positions.device, positions.shape, positions.stride(), inv_freq.dtype, inv_freq.device, inv_freq.shape),
        lambda: _check_rope(what, q, k, q_weight, k_weight, positions, inv_freq, axes))
    dev = q.device
    q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
    q, qs = _heads(q, qs)
    k, ks = _heads(k, ks)
    q_weight, k_weight, inv_freq = _weight(q_weight), _weight(k_weight), inv_freq.contiguous()
    lib = _ext._lib if _ext._lib is not None else load_int4_gemm()
    with _on_device(dev):
        _check(lib.pi05w4a4_qk_norm_rope(q.data_ptr(), qs, k.data_ptr(), ks, *shape, _ptr(q_weight), _ptr(k_weight), eps,
                                         unit_offset, positions.data_ptr(), ps, pos_bytes, count, amap, inv_freq.data_ptr(), rot,
                                         interleaved, q_out.data_ptr(), k_out.data_ptr(), _stream(dev)), "pi05w4a4_qk_norm_rope")
    return q_out, k_out


# ----------------------------------------------------------------------------- custom op
@torch.library.custom_op("pi05_w4a4::qk_norm_rope", mutates_args=())
def _rope_op(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor | None, k_weight: torch.Tensor | None, eps: float,
             positions: torch.Tensor, inv_freq: torch.Tensor, unit_offset: bool, interleaved: bool,
             axes: Sequence[int] | None) -> tuple[torch.Tensor, torch.Tensor]:
    _refuse_tangents(q, k, q_weight, k_weight, inv_freq)
    return _rope_impl(q, k, q_weight, k_weight, eps, positions, inv_freq, unit_offset, interleaved, axes)


@_rope_op.register_fake
def _rope_fake(q, k, q_weight, k_weight, eps, positions, inv_freq, unit_offset, interleaved, axes):
    return q.new_empty(q.shape), k.new_empty(k.shape)


# ----------------------------------------------------------------------------- public functions
def rope_axes(sections: Sequence[int]) -> tuple[int, ...]:
    """The ``axes`` of pairs that stand in runs, ``sections[a]`` of them on axis a: (16, 24, 24) for 64 pairs."""
    return tuple(a for a, n in enumerate(sections) for _ in range(n))


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor | None, k_weight: torch.Tensor | None, eps: float,
                 positions: torch.Tensor, inv_freq: torch.Tensor, unit_offset: bool = True, interleaved: bool = False,
                 axes: Sequence[int] | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Query heads q [B, T, H, D] and key heads k [B, T, KVH, D] (fp16 or bf16, any strides, as the
    parts of a joined QKV product; D a multiple of 16 of at most 512) behind their norm and rotation:
    new contiguous tensors of the same shapes.

    Norm: x / sqrt(mean_d(x^2) + eps) * (unit_offset + weight) of each head, weights [D] in the heads' type;
    None leaves that side without one.  Rotation: pair j turns by positions * inv_freq[j] (fp32 [R / 2], R a
    multiple of 16, R <= D; none for R = 0); it is dimensions (j, j + R / 2), or (2j, 2j + 1) when
    ``interleaved``.  Dimensions from R on are only normed.

    ``positions`` are int32 or int64 [B, T], or [A, B, T] for up to four axes; then ``axes`` (length
    R / 2) names the axis of each pair: ``rope_axes((16, 24, 24))`` for runs, or any order.  fp32
    throughout with one rounding; angles are reduced in 64 bits, so that far positions keep theirs.
    Padding tokens are computed like the others.  There are no derivatives."""
    if _direct(q, k, q_weight, k_weight, positions, inv_freq):
        return _rope_impl(q, k, q_weight, k_weight, float(eps), positions, inv_freq, bool(unit_offset), bool(interleaved), axes)
    return torch.ops.pi05_w4a4.qk_norm_rope(q, k, q_weight, k_weight, float(eps), positions, inv_freq, bool(unit_offset),
                                            bool(interleaved), None if axes is None else list(axes))

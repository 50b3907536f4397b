"""W4A4 (INT4 weight x INT4 activation, Hadamard-rotated) linear layers for MI355X.

Same public names as the reference package ``pi05_fast.w4a4`` (its ``__init__.py:1-11``), and
the 8-bit operators of ``int8`` and ``kv_int8``.
"""

from pi05_fast.w4a4.apply import apply_w4a4_from_dir, maybe_apply_w4a4_from_env
from pi05_fast.w4a4.int8 import add_rms_norm_int8, int8_gemm, quantize_int8, rms_norm_int8
from pi05_fast.w4a4.kv_int8 import int8_kv_append, int8_kv_attention, int8_kv_cache
from pi05_fast.w4a4.linear import W4A4Linear
from pi05_fast.w4a4.pack import int4_gemm_ref, pack_linear_weight

__all__ = [
    "W4A4Linear",
    "apply_w4a4_from_dir",
    "maybe_apply_w4a4_from_env",
    "int4_gemm_ref",
    "pack_linear_weight",
    "quantize_int8",
    "rms_norm_int8",
    "add_rms_norm_int8",
    "int8_gemm",
    "int8_kv_cache",
    "int8_kv_append",
    "int8_kv_attention",
]

"""Limits of the 16-bit serving operators, at the C ABI and without a GPU: workspaces, sizes of a launch, overlaps."""

from __future__ import annotations

import ctypes

import pytest

from pi05_fast.w4a4 import extension as ext

vp = ctypes.c_void_p


@pytest.fixture(scope="module")
def lib():
    return ext.load_int4_gemm()


def _plane(m, r, slices):
    """Bytes of the sums of one K slice: rows in blocks of 16, ranks of a slice in blocks of 32."""
    return (m + 15) // 16 * slices * ((r + 31) // 32) * 512 * 4


@pytest.mark.parametrize("m,per_id", [(16384, 512), (65536, 2048), (65536, 1), (1 << 20, 1 << 15), (1 << 20, 3), (1 << 26, 1 << 26)])
@pytest.mark.parametrize("k,r,slices,adapters", [(16384, 128, 3, 2), (16384, 128, 4, 4), (16384, 16, 1, 9), (1 << 20, 128, 4, 64), (4096, 64, 1, 16)])
def test_sums_of_many_rows(lib, m, per_id, k, r, slices, adapters):
    """However large the adapters are: no more than two planes where rows fill the card, and 256 MB unless one is more."""
    need = lib.pi05w4a4_lora_workspace_bytes(m, per_id, k, 2560, r, slices, adapters)
    plane = _plane(m, r, slices)
    assert plane <= need <= max(plane, min(2 * plane, 1 << 28)) and need % plane == 0


@pytest.mark.parametrize("m", [1, 16, 100, 1197, 3553, 8192])
@pytest.mark.parametrize("k,r,slices,adapters", [(16384, 128, 4, 4), (16384, 8, 4, 300), (1 << 20, 128, 1, 2)])
def test_sums_of_few_rows(lib, m, k, r, slices, adapters):
    assert lib.pi05w4a4_lora_workspace_bytes(m, 1, k, 2560, r, slices, adapters) <= 1 << 27

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


def _lora(lib, m, per_id, n, r=16, adapters=64, y=vp(1 << 45), x=vp(1 << 46), ldx=64, out=vp(1 << 44), ldy=None, ldo=None, ws=None):
    return lib.pi05w4a4_lora_add(y, n if ldy is None else ldy, x, ldx, m, 64, vp(4096), vp(4096), None, adapters, r, vp(4096), per_id, n, 1, None, 0, out,
                                 n if ldo is None else ldo, ws, 0, None)


@pytest.mark.parametrize("m,per_id,n,r", [(1 << 19, 1, 1 << 14, 16), (1 << 18, 1, (1 << 14) + 8, 72), (1 << 22, 3, 1 << 10, 16), (1 << 26, 65, 512, 16)])
def test_adapters_by_rows_have_the_limit_of_whole_tiles(lib, m, per_id, n, r):
    """Windows of many adapters, and requests that end inside a tile, need more workgroups than rows / 16: several launches."""
    assert _lora(lib, m, per_id, n, r) == 3 and b"workspace" in lib.pi05w4a4_last_error()


@pytest.mark.parametrize("m,per_id,n,r", [(1 << 26, 1, 1 << 12, 16), (1 << 26, 3, (1 << 11) + 1, 8), (1 << 20, 1, 1 << 17, 72), (1 << 26, 1 << 26, 1 << 12, 16)])
def test_more_tiles_than_a_launch_holds(lib, m, per_id, n, r):
    assert _lora(lib, m, per_id, n, r) == 1 and b"one launch" in lib.pi05w4a4_last_error()


def test_heads_of_just_too_many_waves(lib):
    """8191 tokens in 8193 parts are 2^26 - 1 waves: in workgroups of four, 2^32 threads."""
    i3 = ctypes.c_int64 * 3
    q, pos, out = vp(1 << 20), vp(4096), vp(1 << 21)
    rc = lib.pi05w4a4_qk_norm_rope(q, i3(512, 512, 512), q, i3(512, 512, 512), 0, 1, 8191, 32767, 16389, 512, None, None, 1e-6, 1, pos,
                                   i3(0, 1, 1), 4, 1, None, pos, 512, 0, out, out, None)
    assert rc == 1 and b"one launch" in lib.pi05w4a4_last_error()


@pytest.mark.parametrize("m,ldy,ldo,at,refused", [
    (2, 32, 32, 0, False), (1, 40, 32, 0, False),  # the output itself
    (2, 40, 32, 0, True), (2, 32, 40, 0, True), (2, 0, 32, 0, True), (1, 32, 32, 2, True), (2, 32, 32, -2, True), (3, 80, 80, 62, True),
    (3, 80, 80, 64, False), (3, 80, 80, -64, False), (3, 80, 80, 160 - 62, True), (2, 32, 32, 128, False), (2, 32, 32, 126, True), (2, 64, 32, -192, False),
])
def test_adapters_read_y_before_they_write_it(lib, m, ldy, ldo, at, refused):
    """y is the output's rows, or apart from them; beside them in wider rows it is apart, and the call fails for its workspace only."""
    rc = lib.pi05w4a4_lora_add(vp((1 << 20) + at), ldy, vp(1 << 24), 16384, m, 16384, vp(4096), vp(4096), None, 2, 8, vp(4096), 1, 32, 1, None, 0,
                               vp(1 << 20), ldo, None, 0, None)
    text = lib.pi05w4a4_last_error()
    assert (rc == 1 and b"y must be" in text) if refused else rc == 3
